// vox_tree_attn.h — attention of the nodes of a draft tree over a ring cache and over their own ancestors.
#pragma once
#include "vox_ops_common.h"

namespace vox {

struct TreeAttnArgs {
    const void *q, *k, *v, *kc, *vc;
    const int *cache_len;
    const uint64_t *ancestors;
    const int *depth;
    void *out;
    float *lse;
    int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, kc_sb, kc_ss, kc_sh, vc_sb, vc_ss, vc_sh, o_sb, o_st, o_sh;   // elements
    int T, H, Hk, G, D, cap, window, W;
    float scale;
};

// First cached position that any node of the sequence may see (depth 0 reaches back furthest) and the cache's length.
__device__ __forceinline__ void tree_range(const TreeAttnArgs &a, int b, int64_t &first, int64_t &len) {
    len = max(a.cache_len[b], 0);
    first = max((int64_t)0, len - a.cap);
    if (a.window > 0) first = max(first, len - a.window + 1);
}

// One workgroup of four waves per (node, head, sequence): a wave takes every fourth key, its lanes split the head's dimensions, and the
// waves' (max, sum, output) are joined at the end.  Any head_dim up to 256, any stride and alignment; a key that is masked is never read.
constexpr int TREE_SCALAR_MAX_D = 256;
template <typename T> __global__ __launch_bounds__(256) void k_tree_attn_scalar(TreeAttnArgs a) {
    __shared__ float sm[4], sl[4], so[4][TREE_SCALAR_MAX_D];
    const int i = blockIdx.x / a.H, h = blockIdx.x - i * a.H, b = blockIdx.y, kvh = h / a.G;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int depth = a.depth[(size_t)b * a.T + i];
    const T *q = (const T *)a.q + b * a.q_sb + i * a.q_st + h * a.q_sh;
    float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) { const int d = lane + 64 * j; qv[j] = d < a.D ? (float)q[d] : 0.f; }
    auto visit = [&](const T *k, const T *v) {
        float dot = 0.f, vv[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = lane + 64 * j;
            vv[j] = d < a.D ? (float)v[d] : 0.f;
            if (d < a.D) dot = fmaf(qv[j], (float)k[d], dot);
        }
        const float s = wave_sum(dot) * a.scale;
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
        const float corr = expf(m - base), p = expf(s - base);
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = o[j] * corr + p * vv[j];
        l = l * corr + p;
        m = mn;
    };
    if (depth >= 0) {
        int64_t first, len;
        tree_range(a, b, first, len);
        if (a.window > 0) first = max(first, len + depth - a.window + 1);
        const T *kc = (const T *)a.kc + b * a.kc_sb + kvh * a.kc_sh, *vc = (const T *)a.vc + b * a.vc_sb + kvh * a.vc_sh;
        for (int64_t p = first + wave; p < len; p += 4) {
            const int64_t slot = p % a.cap;
            visit(kc + slot * a.kc_ss, vc + slot * a.vc_ss);
        }
        const T *kt = (const T *)a.k + b * a.k_sb + kvh * a.k_sh, *vt = (const T *)a.v + b * a.v_sb + kvh * a.v_sh;
        for (int j = wave; j < a.T; j += 4) {
            const bool seen = (a.ancestors[((size_t)b * a.T + i) * a.W + (j >> 6)] >> (j & 63)) & 1;
            if (!seen || (a.window > 0 && a.depth[(size_t)b * a.T + j] <= depth - a.window)) continue;
            visit(kt + j * a.k_st, vt + j * a.v_st);
        }
    }
    if (lane == 0) { sm[wave] = m; sl[wave] = l; }
#pragma unroll
    for (int j = 0; j < 4; j++) so[wave][lane + 64 * j] = o[j];
    __syncthreads();
    const float mm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), base = mm == -INFINITY ? 0.f : mm;
    float f[4], total = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) { f[w] = expf(sm[w] - base); total += f[w] * sl[w]; }
    const int d = threadIdx.x;
    if (d < a.D) {
        float acc = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) acc += f[w] * so[w][d];
        ((T *)a.out)[b * a.o_sb + i * a.o_st + h * a.o_sh + d] = from_f32<T>(total == 0.f ? 0.f : acc / total);
    }
    if (a.lse && threadIdx.x == 0) a.lse[((size_t)b * a.T + i) * a.H + h] = mm + logf(total);
}

}  // namespace vox
