// vox_token_scores.h — rows of logits -> log probabilities of given tokens, entropy, log-sum and the largest logits, in one pass.
//
// Bound by reading the logits once.  A thread keeps the running maximum and sums of its elements, a wave keeps the `top` largest
// elements of its share as a sorted list with one entry per lane, and both are joined over lanes, waves and (few long rows) parts of a row.
#pragma once
#include "vox_ops_common.h"

namespace vox {

// What a pass over some elements leaves, relative to their maximum m:
//   s = sum of e^(x - m) over all of them but ONE that is the maximum (its own term is the 1 of log(1 + s)),
//   t = sum of e^(x - m) (x - m)   (the maximum's own term is 0).
// Then lse = m + log1p(s) and entropy = log1p(s) - t / (1 + s): nothing cancels where one token has almost all the probability.
// No element, or only probability 0: m = -inf, 1 + s = 0.  A NaN among them: m = NaN.
struct RowSum {
    float m, s, t;
};
__device__ __forceinline__ float exp_fast(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896340736f); }
__device__ __forceinline__ RowSum row_join(const RowSum a, const RowSum b) {
    if (a.m != a.m || b.m != b.m) return {NAN, NAN, NAN};
    const bool first = a.m >= b.m;
    const RowSum hi = first ? a : b, lo = first ? b : a;
    if (lo.m == -INFINITY || hi.m == INFINITY) return hi;
    const float d = lo.m - hi.m, f = expf(d), l = 1.f + lo.s;
    return {hi.m, hi.s + f * l, hi.t + f * (lo.t + d * l)};
}

// Orders (value, index) pairs as whole numbers: larger value first, of equal ones (-0 = 0) the lower index.  No pair is 0.  NaN is largest.
__device__ __forceinline__ uint64_t score_key(float x, int index) {
    const unsigned b = __float_as_uint(x + 0.f);
    const unsigned u = x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((uint64_t)u << 32) | (0xffffffffu - (unsigned)index);
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const unsigned u = (unsigned)(key >> 32);
    return u == 0xffffffffu ? NAN : __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_index(uint64_t key) { return (int)(0xffffffffu - (unsigned)key); }

constexpr int SC_TOP = 64, SC_WAVES = 4, SC_THREADS = 64 * SC_WAVES, SC_UNROLL = 4;

struct ScoreArgs {
    const void *logits;
    int64_t row_stride;
    int V, given, top, parts, part_len;      // part_len: elements of a row that one workgroup reads
    const int *tokens;
    float *logprob, *entropy, *lse;
    int *top_index;
    float *top_logprob;
    RowSum *part_sum;                        // [rows, parts]
    uint64_t *part_top;                      // [rows, parts, top]
};

// `n` distinct keys in LDS (0 = none) -> the `top` largest in order: a key's place is the number of larger ones.
__device__ __forceinline__ void top_merge(const uint64_t *keys, int n, int top, uint64_t *out) {
    for (int i = threadIdx.x; i < top; i += SC_THREADS) out[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += SC_THREADS) {
        const uint64_t key = keys[i];
        int place = 0;
        for (int j = 0; j < n; j++) place += keys[j] > key;
        if (key && place < top) out[place] = key;
    }
    __syncthreads();
}

template <typename T> __device__ __forceinline__ void score_finish(const ScoreArgs &a, int64_t row, const RowSum r, const uint64_t *top) {
    const float log1 = log1pf(r.s);
    auto lp = [&](float x) {
        if (r.m != r.m || r.m == INFINITY) return NAN;
        return x == -INFINITY ? -INFINITY : (x - r.m) - log1;
    };
    if (threadIdx.x == 0) {
        const bool none = r.m == -INFINITY;
        a.lse[row] = none || r.m == INFINITY ? r.m : r.m + log1;
        a.entropy[row] = none ? 0.f : r.m == INFINITY ? NAN : log1 - r.t / (1.f + r.s);
    }
    for (int i = threadIdx.x; i < a.given; i += SC_THREADS) {
        const int id = a.tokens[row * a.given + i];
        const bool known = id >= 0 && id < a.V;
        a.logprob[row * a.given + i] = known ? lp((float)((const T *)a.logits)[row * a.row_stride + id]) : r.m != r.m ? NAN : -INFINITY;
    }
    for (int i = threadIdx.x; i < a.top; i += SC_THREADS) {
        a.top_index[row * a.top + i] = key_index(top[i]);
        a.top_logprob[row * a.top + i] = lp(key_value(top[i]));
    }
}

// Grid (rows * parts).  N elements of T per load.
template <typename T, int N> __global__ __launch_bounds__(SC_THREADS) void k_token_scores(ScoreArgs a) {
    __shared__ RowSum sums[SC_WAVES];
    __shared__ uint64_t keys[SC_WAVES * SC_TOP], best[SC_TOP];
    const int64_t row = blockIdx.x / a.parts;
    const int part = blockIdx.x - (int)row * a.parts, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *x = (const T *)a.logits + row * a.row_stride;
    const int begin = part * a.part_len, end = min(begin + a.part_len, a.V);
    RowSum r{-INFINITY, -1.f, 0.f};
    uint64_t list = 0, last = 0;                             // this lane's entry; the list's `top`-th (uniform)
    float bar = NAN;                                         // value of `last` (NaN: the list is not full)
    for (int i0 = begin; i0 < end; i0 += SC_THREADS * N * SC_UNROLL) {
        float f[SC_UNROLL][N];
#pragma unroll
        for (int u = 0; u < SC_UNROLL; u++) {
            const int at = i0 + (u * SC_THREADS + tid) * N;
            if (at + N <= end) load_vec<T, N>(f[u], x + at);
            else
#pragma unroll
                for (int j = 0; j < N; j++) f[u][j] = at + j < end ? (float)x[at + j] : -INFINITY;
        }
#pragma unroll
        for (int u = 0; u < SC_UNROLL; u++) {
            float vm = f[u][0];
#pragma unroll
            for (int j = 1; j < N; j++) vm = fmaxf(vm, f[u][j]);
            if (vm > r.m) {
                const float l = 1.f + r.s, d = r.m - vm, e = r.m == -INFINITY ? 0.f : exp_fast(d);
                r.t = e == 0.f ? 0.f : e * (r.t + d * l);
                r.s = e * l;
                r.m = vm;
                bool own = true;                             // the maximum's own term, once
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const float dj = f[u][j] - vm, ej = exp_fast(dj);
                    if (own && f[u][j] == vm) { own = false; continue; }
                    r.s += ej;
                    r.t += ej * fmaxf(dj, -200.f);           // (e^-inf * -inf is 0 here)
                }
            } else {
                const float base = r.m == -INFINITY ? 0.f : r.m;
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const float dj = f[u][j] - base, ej = exp_fast(dj);
                    r.s += ej;
                    r.t += ej * fmaxf(dj, -200.f);
                }
            }
        }
        if (a.top > 0) {
            // An element that only equals the bar comes behind the elements of earlier trips that put it there: strictly larger ones go on.
            const float limit = bar;
#pragma unroll
            for (int u = 0; u < SC_UNROLL; u++) {
                bool any = false;
#pragma unroll
                for (int j = 0; j < N; j++) any |= !(f[u][j] <= limit);
                if (__ballot(any) == 0) continue;
                const int at = i0 + (u * SC_THREADS + tid) * N;
#pragma unroll
                for (int j = 0; j < N; j++) {
                    uint64_t todo = __ballot(!(f[u][j] <= limit) && at + j < end);
                    const uint64_t mine = score_key(f[u][j], at + j);
                    while (todo) {
                        const int src = __ffsll((unsigned long long)todo) - 1;
                        todo &= todo - 1;
                        const uint64_t key = ((uint64_t)__builtin_amdgcn_readlane((int)(mine >> 32), src) << 32) |
                                             (unsigned)__builtin_amdgcn_readlane((int)mine, src);
                        if (key <= last) continue;
                        const uint64_t above = ((uint64_t)(unsigned)__shfl_up((int)(list >> 32), 1, 64) << 32) | (unsigned)__shfl_up((int)list, 1, 64);
                        list = list > key ? list : (lane == 0 || above > key) ? key : above;
                        last = ((uint64_t)__builtin_amdgcn_readlane((int)(list >> 32), a.top - 1) << 32) |
                               (unsigned)__builtin_amdgcn_readlane((int)list, a.top - 1);
                    }
                }
            }
            bar = last ? key_value(last) : NAN;
        }
    }
    if (r.s != r.s && r.m != INFINITY) r.m = NAN;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const RowSum b{__shfl_xor(r.m, o, 64), __shfl_xor(r.s, o, 64), __shfl_xor(r.t, o, 64)};
        r = row_join(r, b);
    }
    if (lane == 0) sums[wave] = r;
    if (lane < a.top) keys[wave * a.top + lane] = list;
    __syncthreads();
    r = sums[0];
#pragma unroll
    for (int w = 1; w < SC_WAVES; w++) r = row_join(r, sums[w]);
    top_merge(keys, SC_WAVES * a.top, a.top, best);
    if (a.parts == 1) { score_finish<T>(a, row, r, best); return; }
    if (tid == 0) a.part_sum[row * a.parts + part] = r;
    for (int i = tid; i < a.top; i += SC_THREADS) a.part_top[(row * a.parts + part) * a.top + i] = best[i];
}

// Grid (rows): joins the parts of a row.
constexpr int SC_MAX_PARTS = 32;
template <typename T> __global__ __launch_bounds__(SC_THREADS) void k_token_scores_join(ScoreArgs a) {
    __shared__ uint64_t keys[SC_MAX_PARTS * SC_TOP], best[SC_TOP];
    const int64_t row = blockIdx.x;
    for (int i = threadIdx.x; i < a.parts * a.top; i += SC_THREADS) keys[i] = a.part_top[row * a.parts * a.top + i];
    RowSum r = a.part_sum[row * a.parts];
    for (int p = 1; p < a.parts; p++) r = row_join(r, a.part_sum[row * a.parts + p]);
    __syncthreads();
    top_merge(keys, a.parts * a.top, a.top, best);
    score_finish<T>(a, row, r, best);
}

}  // namespace vox
