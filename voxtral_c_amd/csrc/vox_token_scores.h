// vox_token_scores.h — rows of logits -> log probabilities of given tokens, entropy, log-sum and the largest logits, in one pass.
//
// Bound by reading the logits once.  A thread keeps the running maximum and sums of its elements, a wave keeps the `top` largest
// elements of its share as a sorted list with one entry per lane, and both are joined over lanes, waves and (few long rows) parts of a row.
// Measured, vocabulary 131072, on rows that no cache holds: 386 rows of f32, top 4: 49 us (4.1 TB/s; the kernel 43 us, 4.7 TB/s, joining the parts
// 6 us); 1501 rows top 32: bf16 100 us, f16 101 (3.9 TB/s: a 16-bit logit costs the same vector work as an f32 one at half the bytes, and here both count).
// One row, top 8: 7.0 + 5.2 us for parts and join, bound by latency; 12 us a call from Python.
// Rows that do not start on 16 bytes (a contiguous vocabulary that is no multiple of 16 bytes) are read one element per load: 1501 rows of 131071 bf16
// logits 147 us instead of 100, 386 of 131071 f32 63 instead of 49, one row 17 instead of 12.
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
// A distance below -200 counts as -200: its weight e^d is 0 in any case, and 0 times a distance as large as the type's lowest number, or times a sum
// of such, would be NaN.
constexpr float SC_FAR = -200.f;
__device__ __forceinline__ float exp_fast(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896340736f); }
__device__ __forceinline__ RowSum row_join(const RowSum a, const RowSum b) {
    if (a.m != a.m || b.m != b.m) return {NAN, NAN, NAN};
    const bool first = a.m >= b.m;
    const RowSum hi = first ? a : b, lo = first ? b : a;
    if (lo.m == -INFINITY || hi.m == INFINITY) return hi;
    const float d = fmaxf(lo.m - hi.m, SC_FAR), f = expf(d), l = 1.f + lo.s;
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

template <typename T> __device__ __forceinline__ void score_finish(const ScoreArgs &a, int64_t row, const RowSum r, uint64_t list) {
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
    if ((int)threadIdx.x < a.top) {                          // (wave 0 holds the list)
        a.top_index[row * a.top + threadIdx.x] = key_index(list);
        a.top_logprob[row * a.top + threadIdx.x] = lp(key_value(list));
    }
}

__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
    return ((uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}
// A number that at least k of the wave's 64 ordered numbers reach: the k-th largest, bit by bit, to 20 bits.
__device__ __forceinline__ unsigned wave_kth(unsigned v, int k) {
    unsigned t = 0;
#pragma unroll
    for (int bit = 31; bit >= 12; bit--) {
        const unsigned c = t | (1u << bit);
        if (__popcll(__ballot(v >= c)) >= k) t = c;
    }
    return t;
}
__device__ __forceinline__ unsigned ordered(float x) { return (unsigned)(score_key(x, 0) >> 32); }
__device__ __forceinline__ float from_ordered(unsigned u) { return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u); }
// The next larger number (-inf and NaN stay what they are as a bound: nothing is below -inf, and fmaxf passes NaN over).
__device__ __forceinline__ float next_up(float x) { return x == INFINITY || x != x ? x : from_ordered(ordered(x) + 1); }

// The list's lanes one up (lane 0 gets the largest number): v_mov_b32 with wave_shr:1.
__device__ __forceinline__ uint64_t list_above(uint64_t v) {
    const unsigned hi = __builtin_amdgcn_update_dpp(-1, (int)(v >> 32), 0x138, 0xf, 0xf, false);
    const unsigned lo = __builtin_amdgcn_update_dpp(-1, (int)v, 0x138, 0xf, 0xf, false);
    return ((uint64_t)hi << 32) | lo;
}
// The value of lane ^ X: DPP within rows of 16, v_permlane*_swap across them (a fraction of the latency of a trip through ds_bpermute).
template <int X> __device__ __forceinline__ unsigned lane_xor(unsigned v) {
    if constexpr (X == 1) return __builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true);              // quad_perm 1 0 3 2
    else if constexpr (X == 2) return __builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true);         // quad_perm 2 3 0 1
    else if constexpr (X == 4) return __builtin_amdgcn_update_dpp(0, __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true), 0x1B, 0xf, 0xf, true);   // half mirror, quad mirror
    else if constexpr (X == 8) return __builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true);        // row_ror 8
    else if constexpr (X == 15) return __builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true);       // row_mirror
    else if constexpr (X == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (threadIdx.x & 16) ? r[0] : r[1];
    } else {
        static_assert(X == 32, "");
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (threadIdx.x & 32) ? r[0] : r[1];
    }
}
template <int X> __device__ __forceinline__ uint64_t lane_xor64(uint64_t v) {
    return ((uint64_t)lane_xor<X>((unsigned)(v >> 32)) << 32) | lane_xor<X>((unsigned)v);
}
// One step of a bitonic network: of lanes l and l ^ X, the one with bit X clear keeps the larger key if `falling`.
template <int X> __device__ __forceinline__ uint64_t bitonic_step(uint64_t v, bool falling) {
    const uint64_t other = lane_xor64<X>(v);
    return (((threadIdx.x & X) == 0) == falling) == (other > v) ? other : v;
}
template <int X> __device__ __forceinline__ uint64_t bitonic_merge(uint64_t v, bool falling) {
    v = bitonic_step<X>(v, falling);
    if constexpr (X > 1) v = bitonic_merge<X / 2>(v, falling);
    return v;
}
// n keys in the lanes (0 behind them), falling afterwards.
__device__ __forceinline__ uint64_t bitonic_sort(uint64_t v, int n) {
    const int lane = threadIdx.x & 63;
    if (n > 1) v = bitonic_merge<1>(v, (lane & 2) == 0);
    if (n > 2) v = bitonic_merge<2>(v, (lane & 4) == 0);
    if (n > 4) v = bitonic_merge<4>(v, (lane & 8) == 0);
    if (n > 8) v = bitonic_merge<8>(v, (lane & 16) == 0);
    if (n > 16) v = bitonic_merge<16>(v, (lane & 32) == 0);
    if (n > 32) v = bitonic_merge<32>(v, true);
    return v;
}
// The 64 largest of two falling lists, falling.
__device__ __forceinline__ uint64_t list_join(uint64_t list, uint64_t more) {
    more = lane_xor64<32>(lane_xor64<16>(lane_xor64<15>(more)));
    return bitonic_merge<32>(list > more ? list : more, true);
}
// The waves' lists -> wave 0's list; `keys`: [SC_WAVES][64] in LDS.
__device__ __forceinline__ uint64_t waves_join(uint64_t list, uint64_t *keys) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    keys[threadIdx.x] = list;
    __syncthreads();
#pragma unroll
    for (int half = SC_WAVES / 2; half > 0; half >>= 1) {
        if (wave < half) keys[threadIdx.x] = list = list_join(list, keys[(wave + half) * 64 + lane]);
        __syncthreads();
    }
    return list;
}

__device__ __forceinline__ float wave_max_dpp(float v) {
    v = fmaxf(v, __uint_as_float(lane_xor<1>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(lane_xor<2>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(lane_xor<4>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(lane_xor<8>(__float_as_uint(v))));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Grid (rows * parts).  N elements of T per load.  A wave's maximum is one number for all its lanes: it grows about ln(trips) times per row, and
// only then are the sums rescaled (with a maximum per lane, which grows in some
// lane on almost every load, the sums alone took 113 us for 1500 rows of 131072 bf16 logits, with one per wave 80).
template <typename T, int N> __global__ __launch_bounds__(SC_THREADS) void k_token_scores(ScoreArgs a) {
    constexpr int U = N == 8 ? 2 : SC_UNROLL;
    __shared__ RowSum sums[SC_WAVES];
    __shared__ uint64_t pending[SC_WAVES][128];
    // Of each wave's list as it last was: its `top`-th value and its ceil(top / SC_WAVES)-th.  Hints: results do not depend on when they are seen.
    __shared__ float bar_full[SC_WAVES], bar_share[SC_WAVES];
    const int64_t row = blockIdx.x / a.parts;
    const int part = blockIdx.x - (int)row * a.parts, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < SC_WAVES) bar_full[tid] = bar_share[tid] = -INFINITY;
    __syncthreads();
    const T *x = (const T *)a.logits + row * a.row_stride;
    const int begin = part * a.part_len, end = min(begin + a.part_len, a.V);
    float m = -INFINITY, s = 0.f, t = 0.f;                   // RowSum of the wave, s and t by lanes; the maximum's own term is left out of s
    uint64_t *mine = pending[wave];
    uint64_t list = 0, last = 0;                             // this lane's entry; the list's `top`-th (uniform, 0: the list is not full)
    float limit = -INFINITY;                                 // nothing below it can stay
    constexpr int TRIP = SC_THREADS * N * U;
    typedef T vec __attribute__((ext_vector_type(N)));
    vec raw[U];                                      // the next trip's elements, on their way while a trip is worked on
    auto fetch = [&](int i0) {
        if (i0 + TRIP <= end) {
#pragma unroll
            for (int u = 0; u < U; u++) raw[u] = *reinterpret_cast<const vec *>(x + i0 + (u * SC_THREADS + tid) * N);
        }
    };
    fetch(begin);
    for (int i0 = begin; i0 < end; i0 += TRIP) {
        float f[U][N], group[U * N / 4 > 0 ? U * N / 4 : 1], most = -INFINITY;       // group: maxima of four elements each (N = 1: of all)
        if (i0 + TRIP <= end) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < N; j++) f[u][j] = (float)raw[u][j];
        } else {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const int at = i0 + (u * SC_THREADS + tid) * N + j;
                    f[u][j] = at < end ? (float)x[at] : -INFINITY;
                }
        }
        fetch(i0 + TRIP);
#pragma unroll
        for (int g = 0; g < U * N / 4; g++) {
            const int u = g * 4 / N, j = g * 4 % N;          // (N = 1: the four loads)
            group[g] = N >= 4 ? fmaxf(fmaxf(f[u][j], f[u][(j + 1) % N]), fmaxf(f[u][(j + 2) % N], f[u][(j + 3) % N]))
                              : fmaxf(fmaxf(f[u % U][0], f[(u + 1) % U][0]), fmaxf(f[(u + 2) % U][0], f[(u + 3) % U][0]));
            most = fmaxf(most, group[g]);
        }
        const float peak = wave_max_dpp(most);
        if (peak > m) {
            if (m != -INFINITY) {                            // the old maximum's own term joins the others
                const float d = fmaxf(m - peak, SC_FAR), e = exp_fast(d);
                s += lane == 0 ? 1.f : 0.f;
                t = e * (t + d * s);
                s *= e;
            }
            m = peak;
            bool own = (__ffsll((unsigned long long)__ballot(most == peak)) - 1) == lane;      // the new one's, once
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const bool skip = own && f[u][j] == m;
                    const float d = f[u][j] - m, e = skip ? 0.f : exp_fast(d);
                    own = own && !skip;
                    s += e;
                    t += e * fmaxf(d, SC_FAR);               // (e^-inf * -inf is 0 here)
                }
        } else {
            const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const float d = f[u][j] - base, e = exp_fast(d);
                    s += e;
                    t += e * fmaxf(d, SC_FAR);
                }
        }
        if (a.top > 0) {
            // Candidates: what reaches the limit, and NaN, which the sum shows.  The limit comes from this wave's list (strictly above its `top`-th: an
            // equal element of a later trip comes behind it), from the other waves' lists (their `top`-th; and the smallest of all waves'
            // ceil(top / waves)-th, which are `top` elements or more together), and, where many lanes have a candidate, from a number that `top` of
            // the lanes' largest reach.
            const bool nan = __any(s != s);
            if (nan || !(peak < limit)) {
                float all = bar_share[0];
#pragma unroll
                for (int w = 0; w < SC_WAVES; w++) {
                    limit = fmaxf(limit, bar_full[w]);
                    all = fminf(all, bar_share[w]);
                }
                limit = fmaxf(limit, all);
            }
            if (nan || !(peak < limit)) {
                int waiting = 0;                             // keys in `mine` that are not in the list yet
                float here = limit;                          // within this trip (equal elements may still come first)
                const uint64_t lanes = __ballot(nan || !(most < here));
                if (__popcll(lanes) >= max(a.top, 16)) here = fmaxf(here, from_ordered(wave_kth(nan ? 0x007fffffu : ordered(most), a.top)));
#pragma unroll
                for (int g = 0; g < U * N / 4; g++) {
                    if (__ballot(nan || !(group[g] < here)) == 0) continue;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int u = (g * 4 + i) / N, j = (g * 4 + i) % N, at = i0 + (u * SC_THREADS + tid) * N + j;
                        const bool pass = !(f[u][j] < here) && at < end;
                        const uint64_t todo = __ballot(pass);
                        if (todo == 0) continue;
                        if (pass) mine[waiting + __builtin_amdgcn_mbcnt_hi((unsigned)(todo >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)todo, 0))] = score_key(f[u][j], at);
                        waiting += __popcll(todo);
                        if (waiting >= 64) {
                            list = list_join(list, bitonic_sort(mine[lane], 64));
                            waiting -= 64;
                            if (lane < waiting) mine[lane] = mine[64 + lane];
                            last = read_lane(list, a.top - 1);
                            if (last) here = fmaxf(here, key_value(last));
                        }
                    }
                }
                if (waiting > 4) list = list_join(list, bitonic_sort(lane < waiting ? mine[lane] : 0, waiting));
                else
                    for (int i = 0; i < waiting; i++) {      // a few: one by one (a join is nine steps of the network)
                        const uint64_t key = mine[i], above = list_above(list);
                        list = list > key ? list : above > key ? key : above;
                    }
                last = read_lane(list, a.top - 1);
                if (last) {
                    const float bar = key_value(last), share = key_value(read_lane(list, (a.top + SC_WAVES - 1) / SC_WAVES - 1));
                    limit = fmaxf(limit, next_up(bar));
                    if (lane == 0) { bar_full[wave] = bar; bar_share[wave] = share == share ? share : INFINITY; }
                }
            }
        }
    }
    s = wave_sum(s);
    t = wave_sum(t);
    // (an infinite maximum's sum is NaN by itself, inf - inf: only then the wave looks through its elements again)
    bool nan = m != INFINITY && s != s;
    if (m == INFINITY) {
        for (int i0 = begin; i0 < end; i0 += TRIP)
            for (int i = 0; i < U * N; i++) {
                const int at = i0 + (i / N * SC_THREADS + tid) * N + i % N;
                if (at < end && (float)x[at] != (float)x[at]) nan = true;
            }
        nan = __any(nan);
    }
    RowSum r{nan ? NAN : m, m == -INFINITY ? -1.f : s, t};
    if (lane == 0) sums[wave] = r;
    __syncthreads();
    r = sums[0];
#pragma unroll
    for (int w = 1; w < SC_WAVES; w++) r = row_join(r, sums[w]);
    if (a.top > 0) list = waves_join(list, &pending[0][0]);
    if (a.parts == 1) { score_finish<T>(a, row, r, list); return; }
    if (tid == 0) a.part_sum[row * a.parts + part] = r;
    if (tid < a.top) a.part_top[(row * a.parts + part) * a.top + tid] = list;
}

// Grid (rows): joins the parts of a row.
constexpr int SC_MAX_PARTS = 32;
template <typename T> __global__ __launch_bounds__(SC_THREADS) void k_token_scores_join(ScoreArgs a) {
    __shared__ uint64_t pending[SC_WAVES][128];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    RowSum r{-INFINITY, -1.f, 0.f};
    if (lane < a.parts) r = a.part_sum[row * a.parts + lane];
#pragma unroll
    for (int o = 1; o < SC_MAX_PARTS; o <<= 1) {
        const RowSum b{__shfl_xor(r.m, o, 64), __shfl_xor(r.s, o, 64), __shfl_xor(r.t, o, 64)};
        r = row_join(r, b);
    }
    r = RowSum{__shfl(r.m, 0, 64), __shfl(r.s, 0, 64), __shfl(r.t, 0, 64)};
    uint64_t list = 0;
    if (a.top > 0) {
        // The parts' entries number ceil(top / parts) are `top` keys or more together: the smallest of them bounds from below what can stay.
        const uint64_t *keys = a.part_top + row * a.parts * a.top;
        uint64_t bound = lane < a.parts ? keys[lane * a.top + (a.top + a.parts - 1) / a.parts - 1] : ~0ull;
#pragma unroll
        for (int o = 1; o < SC_MAX_PARTS; o <<= 1) {
            const uint64_t b = ((uint64_t)(unsigned)__shfl_xor((int)(bound >> 32), o, 64) << 32) | (unsigned)__shfl_xor((int)bound, o, 64);
            bound = min(bound, b);
        }
        bound = read_lane(bound, 0);
        uint64_t *mine = pending[wave];
        int waiting = 0;
        for (int i = wave * 64; i < a.parts * a.top; i += SC_THREADS) {
            const uint64_t key = i + lane < a.parts * a.top ? keys[i + lane] : 0;
            const bool pass = key && key >= bound;
            const uint64_t todo = __ballot(pass);
            if (pass) mine[waiting + __builtin_amdgcn_mbcnt_hi((unsigned)(todo >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)todo, 0))] = key;
            waiting += __popcll(todo);
            if (waiting >= 64) {
                list = list_join(list, bitonic_sort(mine[lane], 64));
                waiting -= 64;
                if (lane < waiting) mine[lane] = mine[64 + lane];
            }
        }
        if (waiting) list = list_join(list, bitonic_sort(lane < waiting ? mine[lane] : 0, waiting));
        __syncthreads();
        list = waves_join(list, &pending[0][0]);
    }
    score_finish<T>(a, row, r, list);
}

}  // namespace vox
