// k_tree.hip -- what a tree of drafted tokens leaves in the 4-bit KV caches
// (vmlm_hip_tree_accept_kv4).
//
// From token 0 on, the first child that was drafted as the token chosen at its
// parent is the next one; row path[i] of the tree becomes row i. Codes and meta
// move as they are: nothing is quantised again.
//
// A workgroup per (head, sequence, cache) walks the tree again (a ballot a step) rather than
// wait for another's: one launch for up to 16 caches. A row's source never lies before it
// (path[i] >= i), but it may be another's target, so all sources are read, into
// registers (K, meta) and LDS (V: its codes are packed along positions), before the first
// target is written. Bound by latencies: 8 tokens, 2 caches of 36 heads of 64 3.9 us; 16 trees of up to
// 63, 4 such caches 9.3 us.
#include <algorithm>

#include "kv4.hpp"
#include "tree.hpp"

namespace vmlm {
namespace {

constexpr int ACC_THREADS = 256;
constexpr int ACC_BLOCKS = TREE_MAX / KV4_BLOCK + 1;  // blocks that 64 positions touch

struct AcceptParams {
    Kv4Arrays c[TREE_CACHES];
    const int32_t *pos0, *count, *parent, *drafted, *chosen;
    int32_t *path, *kept, *next;  // (null: written by another launch)
    int S, caches, Hkv, cap;
    int *guard;
};

template <int HD>
__global__ __launch_bounds__(ACC_THREADS) void accept_kernel(AcceptParams p) {
    constexpr int NG = HD / 32, T = ACC_THREADS;
    constexpr int KW = TREE_MAX * (HD / 8) / T;   // a thread's dwords of K rows,
    constexpr int MW = (TREE_MAX * NG + T - 1) / T;  // of either meta,
    constexpr int VW = (ACC_BLOCKS * HD + T - 1) / T;  // four of V's blocks
    __shared__ int path[TREE_MAX];
    __shared__ __align__(16) uint32_t vc[ACC_BLOCKS * HD * 4];  // V codes from the first block on
    const int b = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    // 1. the walk, by every wave
    const size_t at = (size_t)b * p.S + min(lane, p.S - 1);
    const int drafted = p.drafted[at], chosen = p.chosen[at];
    const TreeRows t = tree_rows(p.pos0, p.count, p.parent, p.S, p.cap, b, p.guard, h == 0);
    const int n = t.n, pos0 = t.pos0;
    if (n == 0) return;  // an idle sequence
    // (V's blocks are on their way while the tree is walked, whether anything moves or not)
    const Kv4Arrays c = p.c[blockIdx.z];
    const size_t head = (size_t)b * p.Hkv + h, row0 = head * p.cap + pos0;
    const int blk0 = pos0 / KV4_BLOCK, blocks = (pos0 + n - 1) / KV4_BLOCK - blk0 + 1;
    const size_t vat = (head * (p.cap / KV4_BLOCK) + blk0) * (size_t)(HD * 4);
    uint32_t *kd = (uint32_t *)c.k, *vd = (uint32_t *)c.v + vat;
    u32x4 vr[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) {
        const int x = tid + i * T;
        if ((int)blockIdx.z < p.caches && x < blocks * HD) vr[i] = ((const u32x4 *)vd)[x];
    }
    const int parent = p.parent ? t.parent : lane - 1;
    int cur = 0, kept = 1, mine = lane == 0 ? 0 : -1, token;
    int first = 1;  // the first row that moves
    for (;;) {
        token = __builtin_amdgcn_readlane(chosen, cur);
        const unsigned long long hit =
            __ballot(token >= 0 && lane < n && lane > cur && parent == cur && drafted == token);
        if (!hit) break;
        cur = __builtin_ctzll(hit);
        if (lane == kept) mine = cur;
        if (cur == kept && first == kept) ++first;
        ++kept;
    }
    if (p.path && h == 0 && blockIdx.z == 0 && tid < 64) {
        if (lane < p.S) p.path[(size_t)b * p.S + lane] = mine;
        if (lane == 0) {
            p.kept[b] = kept;
            p.next[b] = token;
        }
    }
    if (first >= kept || (int)blockIdx.z >= p.caches) return;
    if (tid < 64) path[lane] = mine;
    // 2. the sources
#pragma unroll
    for (int i = 0; i < VW; ++i)
        if (tid + i * T < blocks * HD) ((u32x4 *)vc)[tid + i * T] = vr[i];
    __syncthreads();
    uint32_t kr[KW], kmr[MW], vmr[MW];
#pragma unroll
    for (int i = 0; i < KW; ++i) {
        const int x = tid + i * T, r = x / (HD / 8);
        if (r >= first && r < kept) kr[i] = kd[(row0 + path[r]) * (HD / 8) + x % (HD / 8)];
    }
#pragma unroll
    for (int i = 0; i < MW; ++i) {
        const int x = tid + i * T, r = x / NG;
        if (r >= first && r < kept) {
            kmr[i] = c.km[(row0 + path[r]) * NG + x % NG];
            vmr[i] = c.vm[(row0 + path[r]) * NG + x % NG];
        }
    }
    __syncthreads();
    // 3. the targets
#pragma unroll
    for (int i = 0; i < KW; ++i) {
        const int x = tid + i * T, r = x / (HD / 8);
        if (r >= first && r < kept) kd[(row0 + r) * (HD / 8) + x % (HD / 8)] = kr[i];
    }
#pragma unroll
    for (int i = 0; i < MW; ++i) {
        const int x = tid + i * T, r = x / NG;
        if (r >= first && r < kept) {
            c.km[(row0 + r) * NG + x % NG] = kmr[i];
            c.vm[(row0 + r) * NG + x % NG] = vmr[i];
        }
    }
    // a dword of V: eight positions of a channel
    const int base = blk0 * KV4_BLOCK - pos0;  // the row of the first block's first position
    for (int i = tid; i < blocks * HD * 4; i += T) {
        const int blk = i / (HD * 4), ch = i / 4 % HD, r0 = base + blk * KV4_BLOCK + i % 4 * 8;
        if (r0 + 7 < first || r0 >= kept) continue;
        uint32_t w = vc[i];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int r = r0 + e;
            if (r < first || r >= kept) continue;
            const int at = path[r] - base;  // from the first block's start
            const uint32_t src = vc[at / KV4_BLOCK * HD * 4 + ch * 4 + at % KV4_BLOCK / 8];
            w = (w & ~(15u << (4 * e))) | (src >> (at % 8 * 4) & 15u) << (4 * e);
        }
        vd[i] = w;
    }
}

}  // namespace

int launch_tree_accept(const AcceptArgs &a, hipStream_t st) {
    for (size_t c0 = 0; c0 == 0 || c0 < a.caches; c0 += TREE_CACHES) {
        AcceptParams p;
        const int n = (int)std::min(a.caches - c0, (size_t)TREE_CACHES);
        for (int i = 0; i < n; ++i) p.c[i] = a.c[c0 + i];
        for (int i = n; i < TREE_CACHES; ++i) p.c[i] = Kv4Arrays{};
        p.pos0 = a.pos0;
        p.count = a.count;
        p.parent = a.parent;
        p.drafted = a.drafted;
        p.chosen = a.chosen;
        p.path = c0 ? nullptr : a.path;
        p.kept = a.kept;
        p.next = a.next;
        p.S = a.S;
        p.caches = n;
        p.Hkv = a.Hkv;
        p.cap = a.cap;
        p.guard = guard_flag_ptr();
        const dim3 grid((unsigned)a.Hkv, (unsigned)a.B, (unsigned)std::max(n, 1));
        switch (a.hd) {
        case 32: accept_kernel<32><<<grid, ACC_THREADS, 0, st>>>(p); break;
        case 64: accept_kernel<64><<<grid, ACC_THREADS, 0, st>>>(p); break;
        case 128: accept_kernel<128><<<grid, ACC_THREADS, 0, st>>>(p); break;
        default: accept_kernel<256><<<grid, ACC_THREADS, 0, st>>>(p); break;
        }
        VMLM_HIP_CHECK(hipGetLastError());
    }
    return VMLM_OK;
}

}  // namespace vmlm
