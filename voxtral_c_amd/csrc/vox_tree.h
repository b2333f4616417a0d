// vox_tree.h — draft trees: ancestor sets, acceptance, and the accepted rows' way into the ring cache.
// All three are bound by the latency of a launch and of one to three dependent trips to memory; a tree has at most 256 nodes, so one workgroup
// with a thread per node holds all of it and every step is a constant number of barriers.  Measured, plan / accept / commit: one tree of 2
// nodes, 26 layers of 8 x 128 f32: 1.4 / 2.4 / 3.4 us; 8 trees of 63 nodes in bf16: 3.4 / 3.5 / 3.6 us.  The three calls from Python take 15.6 us: the host
// is the bound (three launches are 10 of them).
#pragma once
#include "vox_ops_common.h"

namespace vox {

constexpr int TREE_MAX = 256, TREE_WORDS = TREE_MAX / 64;

// Ancestor sets by pointer doubling: anc(i) = {i}, jump(i) = parent(i); a round makes anc(i) |= anc(jump(i)), jump(i) = jump(jump(i)),
// after which anc(i) holds the nearest 2^round nodes of the chain: ceil(log2 nodes) rounds instead of a walk of up to 255 steps.
__global__ __launch_bounds__(TREE_MAX) void k_tree_plan(const int *parents, const int *n_nodes, int T, uint64_t *ancestors, int *depth) {
    __shared__ uint64_t anc[TREE_MAX][TREE_WORDS];
    __shared__ int jump[TREE_MAX];
    __shared__ int cut[TREE_MAX];
    const int b = blockIdx.x, i = threadIdx.x, W = (T + 63) >> 6;
    const int n = n_nodes ? min(max(n_nodes[b], 0), T) : T;
    const int p = i < T ? parents[(size_t)b * T + i] : -1;
    const bool ok = i < n && p >= -1 && p < i;
    uint64_t a[TREE_WORDS];
#pragma unroll
    for (int w = 0; w < TREE_WORDS; w++) { a[w] = (i >> 6) == w ? 1ull << (i & 63) : 0ull; anc[i][w] = a[w]; }
    int j = ok ? p : -1, c = ok ? 0 : 1;
    jump[i] = j; cut[i] = c;
    __syncthreads();
    for (int span = 1; span < T; span <<= 1) {
        int jj = -1;
        if (j >= 0) {
#pragma unroll
            for (int w = 0; w < TREE_WORDS; w++) a[w] |= anc[j][w];
            c |= cut[j];
            jj = jump[j];
        }
        __syncthreads();
        j = jj;
#pragma unroll
        for (int w = 0; w < TREE_WORDS; w++) anc[i][w] = a[w];
        jump[i] = j; cut[i] = c;
        __syncthreads();
    }
    if (i >= T) return;
    int d = -1;
#pragma unroll
    for (int w = 0; w < TREE_WORDS; w++) {
        if (w >= W) break;
        ancestors[((size_t)b * T + i) * W + w] = c ? 0ull : a[w];
        d += __popcll(a[w]);
    }
    depth[(size_t)b * T + i] = c ? -1 : d;
}

// A node matches if its token is the choice behind its parent; of matching siblings (they all carry the same token) the lowest
// index stays.  A node is accepted if all its ancestors and itself match: anc(i) & ~match = 0.  The accepted nodes form one chain, so
// a node's place in the path is its depth.
__global__ __launch_bounds__(TREE_MAX) void k_tree_accept(const int *tokens, const int *choices, const int *root_choice, const int *parents,
                                                          const uint64_t *ancestors, const int *depth, const int *cache_len, int T, int *path,
                                                          int *n_accepted, int *next_token, int *new_len) {
    __shared__ int first[TREE_MAX + 1];
    __shared__ int line[TREE_MAX];
    __shared__ uint64_t match[TREE_WORDS];
    const int b = blockIdx.x, i = threadIdx.x, W = (T + 63) >> 6;
    const size_t row = (size_t)b * T;
    first[i] = TREE_MAX;
    if (i == 0) first[TREE_MAX] = TREE_MAX;
    const int d = i < T ? depth[row + i] : -1;
    const int p = i < T ? parents[row + i] : -2;
    const bool there = d >= 0 && d < T && p >= -1 && p < T;
    const int want = p >= 0 && p < T ? choices[row + p] : root_choice[b];
    const bool m = there && tokens[row + i] == want;
    uint64_t a[TREE_WORDS];
#pragma unroll
    for (int w = 0; w < TREE_WORDS; w++) a[w] = i < T && w < W ? ancestors[(row + i) * W + w] : 0ull;
    __syncthreads();
    if (m) atomicMin(&first[p + 1], i);
    __syncthreads();
    const uint64_t bits = __ballot(m && first[p + 1] == i);
    if ((i & 63) == 0) match[i >> 6] = bits;
    line[i] = -1;
    __syncthreads();
    bool ok = m && ((match[i >> 6] >> (i & 63)) & 1);
#pragma unroll
    for (int w = 0; w < TREE_WORDS; w++) ok = ok && (a[w] & ~match[w]) == 0;
    if (ok) line[d] = i;
    const int count = __syncthreads_count(ok);
    if (i < T) path[row + i] = line[i];
    if (i == 0) {
        const int last = count > 0 ? line[count - 1] : -1;      // (-1 behind a node only where the masks are no tree's)
        next_token[b] = last >= 0 ? choices[row + last] : root_choice[b];
        n_accepted[b] = count;
        new_len[b] = max(cache_len[b], 0) + count;
    }
}

struct TreeCommitArgs {
    const char *k, *v;
    char *kc, *vc;
    int64_t k_s[4], v_s[4], kc_s[4], vc_s[4];       // bytes: layer, batch, row, head
    const int *path, *n_accepted, *cache_len;
    int T, Hk, head_bytes, cap;
};
// Accepted rows to their ring slots, V bytes per access.  Grid: (batch, layers x {k, v}, groups of COMMIT_ROWS path entries).
constexpr int COMMIT_ROWS = 8;
template <typename V> __global__ __launch_bounds__(256) void k_tree_commit(TreeCommitArgs a) {
    const int b = blockIdx.x, layer = blockIdx.y >> 1, j0 = blockIdx.z * COMMIT_ROWS;
    const int n = min(a.n_accepted[b], a.T);
    if (j0 >= n) return;
    const bool is_v = blockIdx.y & 1;
    const char *src = (is_v ? a.v : a.k) + layer * (is_v ? a.v_s[0] : a.k_s[0]) + b * (is_v ? a.v_s[1] : a.k_s[1]);
    char *dst = (is_v ? a.vc : a.kc) + layer * (is_v ? a.vc_s[0] : a.kc_s[0]) + b * (is_v ? a.vc_s[1] : a.kc_s[1]);
    const int64_t sr = is_v ? a.v_s[2] : a.k_s[2], sh = is_v ? a.v_s[3] : a.k_s[3];
    const int64_t dr = is_v ? a.vc_s[2] : a.kc_s[2], dh = is_v ? a.vc_s[3] : a.kc_s[3];
    const int64_t len = max(a.cache_len[b], 0);
    const int per_head = a.head_bytes / (int)sizeof(V), per_row = per_head * a.Hk;
    const int rows = min(n - j0, COMMIT_ROWS);
    for (int t = threadIdx.x; t < rows * per_row; t += 256) {
        const int r = t / per_row, e = t - r * per_row, h = e / per_head, x = e - h * per_head;
        const int node = a.path[(size_t)b * a.T + j0 + r];
        if (node < 0 || node >= a.T) continue;
        const int64_t slot = (len + j0 + r) % a.cap;
        *reinterpret_cast<V *>(dst + slot * dr + h * dh + (int64_t)x * sizeof(V)) =
            *reinterpret_cast<const V *>(src + node * sr + h * sh + (int64_t)x * sizeof(V));
    }
}

}  // namespace vox
