// vox_tree_attn.h — attention of the nodes of a draft tree over a ring cache and over their own ancestors.
#pragma once
#include <type_traits>
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
// waves' (max, sum, output) are joined at the end.  Any head_dim up to 256, any stride and alignment; a key that is masked is never read.  Bound by the latency
// of one key after another, each read again for every node and head: 2 nodes x 32 heads of 33 dimensions over 8192 keys, f32: 1.56 ms; 4 x 4 nodes x 32 heads of
// 100, bf16: 3.4 ms, where 104 dimensions (rows of whole 16-byte loads) take 37 us.  It is there so that every layout is answered, not for speed.
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


// ---- matrix-pipe form ----------------------------------------------------------------------------------------------------------
// The G query heads of a kv head share its keys, so the rows of a (sequence, kv head) are its nodes x G heads, taken in tiles of 16.  KT keys
// are a step, and both products are transposed so that the weights never leave their registers:
//   S^T[key, row] = K . Q^T      K is the A operand (lane: key = lane % 16, its share of the head's dimensions), Q^T stays in registers;
//   O^T[d, row]  += V^T . P^T    the lane that holds S^T's column (row = lane % 16) for keys 4 c + r, c = lane / 16, holds exactly
//                                what the B operand wants of P^T if the product's inner index runs over keys in that order, and V is read as the
//                                A operand in the same order: lane m of a 16-lane row takes VU consecutive dimensions (16 m VU ..) of the keys
//                                4 c + r and supplies one of them to each of E products.
// Two ways to the keys:
//   own      (up to 16 rows, 32 where a head has up to 64 dimensions) every wave has keys of its own, straight from memory into the registers that the
//            matrix instruction reads, 16 bytes per lane; K of the next step is requested when the scores are done, V when the outputs are.  Bound by
//            the read of the cache, and for short caches by latency: 2 nodes x 4 heads over 232 keys, f32: 11.2 us, the join of 4 parts 3.9 us.
//   shared   (more rows) the four waves have rows of their own and share the steps' keys in LDS, which global_load_lds fills STAGES steps ahead:
//            nothing of it is in registers, and the cache is read once per 64 or 128 rows.  24 nodes x 4 heads over 4 x 40000 keys, bf16: 127 us for 557 MB
//            (4.4 TB/s), bound by the read; 64 nodes x 4 heads over 2 x 8191 keys, f32: 174 us, bound by the vector unit, which splits the numbers (below).
// Where both would do, 32 rows of 128 dimensions over 4 x 16000 keys: own 78 us, shared 57 in bf16, 152 and 125 in f32.
// Head sizes between 64, 128 and 256 run as the next one of these, and none of their tiles is plain (below): 96 dimensions, 24 nodes x 4 heads over 4 x 40000
// keys, bf16: 130 us for 418 MB, 3.2 TB/s; 2 nodes x 4 heads: 97 us, 4.3 TB/s (128 dimensions: 115 us, 4.9 TB/s).
// Each wave runs its own online softmax (one maximum and sum per row); waves with different keys are joined through LDS at the end, the parts of a
// long cache by k_tree_attn_join.
template <typename T> struct AttnType;
template <> struct AttnType<float> {
    static constexpr int SHIFT = 0;
    typedef unsigned Bits;
    static constexpr Bits INF = 0x7f800000u, SIGN = 0x80000000u;
    static constexpr float LAZY = 8.f;
};
// P is rounded to bf16 in front of its product (a half step of 2^-8 per weight, like the rounding of the output itself): the product then runs at
// the 16-bit rate.  The weights' sum is taken of the f32 values.
template <> struct AttnType<bf16_t> {
    static constexpr int SHIFT = 0;
    typedef unsigned short Bits;
    static constexpr Bits INF = 0x7f80, SIGN = 0x8000;
    static constexpr float LAZY = 8.f;
};
// f16: the same with a half step of 2^-11; weights are lifted by 2^12 so that what is 2^-26 of the largest one is still a normal number (a sum over
// tens of thousands of small weights would lose them otherwise).
template <> struct AttnType<f16_t> {
    static constexpr int SHIFT = 12;
    typedef unsigned short Bits;
    static constexpr Bits INF = 0x7c00, SIGN = 0x8000;
    static constexpr float LAZY = 3.f;
};

constexpr int ATTN_WAVES = 4;
// Shared keys of f32 are multiplied on the bf16 pipe: a number is exactly the sum of three bf16 ones (8 of its 24 bits each, cut off, so all of its sign),
// and of the nine products six are taken.  With the leading bit as 1 the middle part is below 2^-7 and the low one below 2^-15: the two products of a
// middle and a low part that are left out are up to 2^-21 of the whole product together (2^-21.03 for 1 + 2^-7 - 2^-23 squared; 2^-24.5 on average
// over normally distributed numbers), always with its sign.  An f32 matrix instruction takes the vector unit's cycles (measured:
// the two run one after the other, 0.23 + 0.23 ms -> 0.46 ms), a bf16 one does not, and six of them take 6 x 17 cycles where f32 takes 8 x 33:
// 64 rows over 4 x 16000 keys 163 -> 142 us, 32 rows 152 -> 125.  Splitting each key once per workgroup into LDS, by eight waves in step, was slower at
// 64 rows (178 us instead of 142) and faster above (128 rows 239 instead of 267, 256 rows 432 instead of 481); there is one form for all of them.
template <typename T, bool SHARED> constexpr bool ATTN_SPLIT = SHARED && sizeof(T) == 4;
template <typename T, bool SHARED> constexpr int ATTN_KT = SHARED || sizeof(T) == 2 ? 32 : 16;              // keys of a step
template <typename T> constexpr int ATTN_STAGES = sizeof(T) == 4 ? 2 : 3;                                   // (two workgroups per CU)
struct TreeAttnPlan {
    int splits, row_blocks;
    float *part_o, *part_ml;      // [splits][batch * Hk][rows][D], [splits][batch * Hk][rows][2]
};

__device__ __forceinline__ float max_over_c(float v) {        // over lanes l, l ^ 16, l ^ 32, l ^ 48
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_over_c(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// One step of 16 x 16 outputs: an inner index of 32 (16-bit types, 8 values per lane) or 16 (f32: four instructions of 4).
template <typename T, typename V> __device__ __forceinline__ f32x4 attn_mma(const V x, const V y, f32x4 acc) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], acc, 0, 0, 0);
        return acc;
    } else if constexpr (__is_same(T, bf16_t)) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, acc, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, acc, 0, 0, 0);
}

// Eight numbers of f32 as three bf16 operands: x = h + m + l exactly (each step takes the number's top 8 bits and leaves the rest).
template <typename V, typename F> __device__ __forceinline__ void split3(F x, V &h, V &m, V &l) {
    typedef unsigned words __attribute__((ext_vector_type(4)));
    words hw, mw, lw;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = x(2 * i), b = x(2 * i + 1);
        hw[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);          // the upper halves of b and a
        const float a1 = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u), b1 = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
        mw[i] = __builtin_amdgcn_perm(__float_as_uint(b1), __float_as_uint(a1), 0x07060302u);
        const float a2 = a1 - __uint_as_float(__float_as_uint(a1) & 0xffff0000u), b2 = b1 - __uint_as_float(__float_as_uint(b1) & 0xffff0000u);
        lw[i] = __builtin_amdgcn_perm(__float_as_uint(b2), __float_as_uint(a2), 0x07060302u);
    }
    h = __builtin_bit_cast(V, hw);
    m = __builtin_bit_cast(V, mw);
    l = __builtin_bit_cast(V, lw);
}
// acc + x y of split numbers, smallest products first.
template <typename V> __device__ __forceinline__ f32x4 split_mma(const V (&x)[3], const V (&y)[3], f32x4 acc) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[2], y[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[0], y[2], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[1], y[1], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[1], y[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[0], y[1], acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[0], y[0], acc, 0, 0, 0);
}

// Key tiles of a sequence: the cache's, then the tree's; split s takes tiles [s * per, (s + 1) * per).
struct TileRange {
    int64_t first, len;
    int cached, n_cache, n_all, per;
};
template <int KT> __device__ __forceinline__ TileRange tile_range(const TreeAttnArgs &a, int b, int splits, int key_waves) {
    TileRange r;
    tree_range(a, b, r.first, r.len);
    r.cached = (int)(r.len - r.first);
    r.n_cache = (int)(((int64_t)r.cached + KT - 1) / KT);
    r.n_all = r.n_cache + (a.T + KT - 1) / KT;
    r.per = ((r.n_all + splits - 1) / splits + key_waves - 1) / key_waves * key_waves;
    return r;
}

// One tile's keys: row `base`, key i in row base + (i < wrap ? i : i - cap), `count` of them.
struct KeyTile {
    const char *k, *v;
    int ks, vs;                   // bytes between rows
    int count, wrap, cap;
};

// Bytes of LDS of a workgroup: the stages (shared) or Q^T (own, where registers do not hold it), later the outputs; and maxima and sums.
template <typename T, int DP, int RT, bool SHARED> constexpr int attn_lds() {
    const int rows = RT * 16 * (SHARED ? ATTN_WAVES : 1), out = rows * (DP + 4) * 4, stages = SHARED ? ATTN_STAGES<T> * 2 * ATTN_KT<T, SHARED> * DP * (int)sizeof(T) : 0;
    return (out > stages ? out : stages) + 2 * (SHARED ? 1 : ATTN_WAVES) * rows * 4;
}

template <typename T, int DP, int RT, bool SHARED>
__global__ __launch_bounds__(64 * ATTN_WAVES, (DP == 256 || (ATTN_SPLIT<T, SHARED> && DP * RT > 128) ? 1 : 2)) void k_tree_attn(TreeAttnArgs a, TreeAttnPlan plan) {
    typedef AttnType<T> A;
    typedef typename A::Bits bits_t;
    constexpr bool SPLIT = ATTN_SPLIT<T, SHARED>;
    constexpr int KT = ATTN_KT<T, SHARED>, STAGES = ATTN_STAGES<T>, E = DP / 16, NK = KT / 16, VK = KT / 4;      // VK: keys per lane of a V operand
    constexpr int U = sizeof(T) == 2 ? 8 : 4;                                    // elements per 16-byte load
    constexpr int KS = DP / (4 * U);                                             // K / Q loads per lane and 16 keys / rows
    typedef typename std::conditional<SPLIT, bf16_t, T>::type M;                 // what the matrix instructions take, MU values per lane
    constexpr int MU = sizeof(M) == 2 ? 8 : 4, MS = DP / (4 * MU);               // MS: steps over the dimensions
    typedef M mvec __attribute__((ext_vector_type(MU)));
    constexpr int VU = E < U ? E : U, VL = E / VU;                               // V: VL loads of VU elements per key
    constexpr float LOG2E = 1.44269504088896340736f;
    typedef T kvec __attribute__((ext_vector_type(U)));
    typedef T vvec __attribute__((ext_vector_type(VU)));
    constexpr int RW = SHARED ? ATTN_WAVES : 1, KW = ATTN_WAVES / RW;            // waves side by side over rows, over keys
    constexpr int WROWS = RT * 16, ROWS = WROWS * RW, LD = DP + 4;               // rows of a wave, of the workgroup
    extern __shared__ __attribute__((aligned(128))) char lds[];
    float *so = reinterpret_cast<float *>(lds);                                  // [ROWS][LD]: the outputs, one key wave's after another's
    float *sm = reinterpret_cast<float *>(lds + attn_lds<T, DP, RT, SHARED>()) - 2 * KW * ROWS, *sl = sm + KW * ROWS;        // [KW][ROWS] each

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n16 = lane & 15, c = lane >> 4;
    // Workgroups that read the same keys (the row blocks of a group) have numbers that differ by 8: they land on one XCD and share its L2.
    const int RB = plan.row_blocks, chunk = blockIdx.x / (8 * RB), in = blockIdx.x - chunk * 8 * RB;
    const int group = chunk * 8 + (in & 7), rb = in >> 3;
    const int b = blockIdx.y, split = group / a.Hk, kvh = group - split * a.Hk;
    if (split >= plan.splits) return;
    const int R = a.T * a.G, row0 = rb * ROWS;
    const int kw = SHARED ? 0 : wave, rw = SHARED ? (wave + split) & (ATTN_WAVES - 1) : 0;       // (idle waves on another SIMD from split to split)
    const int wrow0 = row0 + rw * WROWS;
    const bool idle = wrow0 >= R;                            // (the last workgroup's waves behind the last row)

    // this lane's query rows, requested in front of the cache's length; a negative scale goes into Q's sign
    constexpr bool QLDS = !SHARED && (sizeof(T) == 4 || DP == 256);
    mvec qf[QLDS ? 1 : RT][QLDS ? 1 : MS][SPLIT ? 3 : 1];
    kvec *qs = reinterpret_cast<kvec *>(lds);                // [RT][KS][64 lanes]
    kvec qr[RT][KS];
    int row_depth[RT], row_node[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const int row = wrow0 + t * 16 + n16, node = row < R ? row / a.G : 0, h = kvh * a.G + (row - node * a.G);
        row_node[t] = node;
        row_depth[t] = row < R ? min(a.depth[(size_t)b * a.T + node], 1 << 30) : -1;
        const T *q = (const T *)a.q + b * a.q_sb + node * a.q_st + h * a.q_sh;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            // (a matrix operand takes MU values in a row: two of f32's loads, where it is split)
            const int d = SPLIT ? (i >> 1) * 4 * MU + c * MU + (i & 1) * U : i * 4 * U + c * U;
            qr[t][i] = kvec(T(0.f));
            if (row < R && d < a.D && (!QLDS || kw == 0)) qr[t][i] = *reinterpret_cast<const kvec *>(q + d);
        }
    }
    const TileRange tr = tile_range<KT>(a, b, plan.splits, KW);
    const int t_begin = split * tr.per, t_end = min(t_begin + tr.per, tr.n_all);
    if (t_begin >= t_end) return;
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int i = 0; i < KS; i++)
            if (a.scale < 0.f) qr[t][i] = -qr[t][i];
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int s = 0; s < MS; s++) {
            if constexpr (SPLIT) split3<mvec>([&](int i) { return qr[t][s * 2 + (i >> 2)][i & 3]; }, qf[t][s][0], qf[t][s][1], qf[t][s][2]);
            else if constexpr (!QLDS) qf[t][s][0] = qr[t][s];
            else if (kw == 0) qs[(t * KS + s) * 64 + lane] = qr[t][s];
        }
    const float scale2 = fabsf(a.scale) * LOG2E;

    const char *kc = (const char *)((const T *)a.kc + b * a.kc_sb + kvh * a.kc_sh), *vc = (const char *)((const T *)a.vc + b * a.vc_sb + kvh * a.vc_sh);
    const int ks = (int)a.kc_ss * (int)sizeof(T), vs = (int)a.vc_ss * (int)sizeof(T);            // (less than 2^26: attn_wide)
    const unsigned slot_first = (unsigned)(tr.first % a.cap);
    auto slot_of = [&](int t) {
        const unsigned slot = slot_first + (unsigned)t * KT;
        return slot >= (unsigned)a.cap ? slot - a.cap : slot;
    };
    // Tiles [full_begin, full_end) are seen whole by every row of the workgroup: behind the window's edge of its deepest one, in front of the cache's
    // end.  A tile of
    // those that the ring does not break is plain: its rows follow each other, and a lane's offsets within it are the same for every tile.
    const int edge = (int)max(tr.len + 1 - a.window - tr.first, (int64_t)-(1 << 30));            // first position of a window at depth 0, from `first`
    const int full_end = tr.cached / KT;
    int deepest = 0, full_begin = 0;                         // (behind the first tiles' loads)
    auto is_masked = [&](int t) { return t < full_begin || t >= full_end; };
    auto is_plain = [&](int t) { return a.D == DP && t < full_end && slot_of(t) + KT <= (unsigned)a.cap; };
    auto tile_at = [&](int t) {
        KeyTile x;
        if (t < tr.n_cache) {
            const int64_t slot = slot_of(t);
            x.k = kc + slot * ks;
            x.v = vc + slot * vs;
            x.ks = ks;
            x.vs = vs;
            x.count = min(KT, tr.cached - t * KT);
            x.wrap = (int)min((int64_t)KT, a.cap - slot);
        } else {
            const int off = (t - tr.n_cache) * KT;
            x.k = (const char *)((const T *)a.k + b * a.k_sb + kvh * a.k_sh + off * a.k_st);
            x.v = (const char *)((const T *)a.v + b * a.v_sb + kvh * a.v_sh + off * a.v_st);
            x.ks = (int)a.k_st * (int)sizeof(T);
            x.vs = (int)a.v_st * (int)sizeof(T);
            x.count = min(KT, a.T - off);
            x.wrap = KT;
        }
        x.cap = a.cap;
        return x;
    };
    // Which of a tile's keys (bit i) does row tile r's row of this lane see?
    auto visible = [&](int t, int count, int r) {
        unsigned bits = 0xffffffffu;
        if (t >= tr.n_cache) {
            const int off = (t - tr.n_cache) * KT;
            bits = (unsigned)(a.ancestors[((size_t)b * a.T + row_node[r]) * a.W + (off >> 6)] >> (off & 63));
            if (a.window > 0) {
                const int d = (lane & 31) < count ? a.depth[(size_t)b * a.T + off + (lane & 31)] : 0x7fffffff;
                if (__any(d <= deepest - a.window))          // (only trees that are deeper than the window)
                    for (int j = 0; j < count; j++)
                        if (__builtin_amdgcn_readlane(d, j) <= row_depth[r] - a.window) bits &= ~(1u << j);
            }
        } else if (a.window > 0) {
            const int below = edge + row_depth[r] - t * KT;  // keys in front of the row's window
            bits = below >= 32 ? 0u : below <= 0 ? 0xffffffffu : 0xffffffffu << below;
        }
        return count < 32 ? bits & ((1u << count) - 1u) : bits;
    };
    auto bits_of = [](T x) { return __builtin_bit_cast(bits_t, x); };

    // ---- keys of the wave's own
    kvec kf[SHARED ? 1 : NK][SHARED ? 1 : KS];
    vvec vf[VK][VL];
    auto load_k = [&](int t) {
        if constexpr (!SHARED) {
            if (is_plain(t)) {
                const char *base = kc + (int64_t)slot_of(t) * ks;
#pragma unroll
                for (int i = 0; i < NK; i++)
#pragma unroll
                    for (int s = 0; s < KS; s++) kf[i][s] = *reinterpret_cast<const kvec *>(base + ((unsigned)((i * 16 + n16) * ks + c * 16) + s * 64));
                return;
            }
            const KeyTile x = tile_at(t);
#pragma unroll
            for (int i = 0; i < NK; i++) {
                const int key = i * 16 + n16, row = key < x.wrap ? key : key - x.cap;
                const T *p = reinterpret_cast<const T *>(x.k + (int64_t)row * x.ks);
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    const int d = s * 4 * U + c * U;
                    if (key < x.count && d < a.D) kf[i][s] = *reinterpret_cast<const kvec *>(p + d);
                    else kf[i][s] = kvec(T(0.f));
                }
            }
        }
    };
    auto load_v = [&](int t) {
        if (!SHARED && is_plain(t)) {
            const char *base = vc + (int64_t)slot_of(t) * vs;
#pragma unroll
            for (int j = 0; j < VK; j++)
#pragma unroll
                for (int u = 0; u < VL; u++)
                    vf[j][u] = *reinterpret_cast<const vvec *>(base + ((unsigned)(((j >> 2) * 16 + c * 4 + (j & 3)) * vs + n16 * VU * (int)sizeof(T)) + u * 16 * VU * (int)sizeof(T)));
            return;
        }
        const KeyTile x = tile_at(t);
#pragma unroll
        for (int j = 0; j < VK; j++) {
            const int key = (j >> 2) * 16 + c * 4 + (j & 3), row = key < x.wrap ? key : key - x.cap;
            const T *p = reinterpret_cast<const T *>(x.v + (int64_t)row * x.vs);
#pragma unroll
            for (int u = 0; u < VL; u++) {
                const int d = (u * 16 + n16) * VU;
                if (key < x.count && d < a.D) vf[j][u] = *reinterpret_cast<const vvec *>(p + d);
                else vf[j][u] = vvec(T(0.f));
            }
        }
    };

    // ---- keys in LDS: per stage K [KT][DP], V [KT][DP]; 16-byte piece q of row r sits at q ^ swizzle(r): 16 lanes of an access (16 rows, one piece each)
    // touch every one of the 64 banks once
    constexpr int PIECES = DP * (int)sizeof(T) / 16, TILE = KT * DP * (int)sizeof(T), LOADS = TILE / (1024 * ATTN_WAVES);        // LOADS: per wave, for K and for V
    static_assert(TILE % (1024 * ATTN_WAVES) == 0, "a tile is a whole number of a workgroup's loads");
    auto swizzle = [](int row) { return PIECES >= 16 ? row & 15 : (row >> 1) & 7; };
    auto piece_at = [&](int row, int q) { return (row * PIECES + (q ^ swizzle(row))) * 16; };
    auto issue = [&](int t, int stage) {
        const unsigned base = lds_addr(lds) + (unsigned)stage * (2 * TILE);
        if (is_plain(t)) {
            const char *k = kc + (int64_t)slot_of(t) * ks, *v = vc + (int64_t)slot_of(t) * vs;
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const int at = (i * ATTN_WAVES + wave) * 64, row = (at + lane) / PIECES, q = ((at + lane) % PIECES) ^ swizzle(row);
                glds16_at(k, (unsigned)(row * ks + q * 16), __builtin_amdgcn_readfirstlane(base + at * 16));
                glds16_at(v, (unsigned)(row * vs + q * 16), __builtin_amdgcn_readfirstlane(base + TILE + at * 16));
            }
            return;
        }
        const KeyTile x = tile_at(t);
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int at = (i * ATTN_WAVES + wave) * 64, row = (at + lane) / PIECES, q = ((at + lane) % PIECES) ^ swizzle(row), from = row < x.wrap ? row : row - x.cap;
            if (row < x.count && q * U < a.D) {
                glds16(x.k + (int64_t)from * x.ks + q * 16, __builtin_amdgcn_readfirstlane(base + at * 16));
                glds16(x.v + (int64_t)from * x.vs + q * 16, __builtin_amdgcn_readfirstlane(base + TILE + at * 16));
            }
        }
    };

    auto read_v = [&](const char *sv, int from, int to) {
#pragma unroll
        for (int j = 0; j < VK; j++) {
            const int key = (j >> 2) * 16 + c * 4 + (j & 3);
#pragma unroll
            for (int u = 0; u < VL; u++) {
                const int at = (u * 16 + n16) * VU * (int)sizeof(T);             // byte of the row
                if (u >= from && u < to) vf[j][u] = *reinterpret_cast<const vvec *>(sv + piece_at(key, at >> 4) + (at & 15));
            }
        }
    };

    f32x4 o[RT][E];
    float m[RT], l[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        m[t] = -INFINITY; l[t] = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) o[t][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bool bad = false;                                        // a masked tile held a value that is not finite

    int t = SHARED ? t_begin : t_begin + kw, stage = 0;
    if constexpr (SHARED) {
        if (a.D < DP) {                                      // dimensions that no load fills
            for (int i = tid; i < STAGES * 2 * TILE / 16; i += 64 * ATTN_WAVES) reinterpret_cast<uint4 *>(lds)[i] = uint4{0, 0, 0, 0};
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++)
            if (t + i < t_end) issue(t + i, i);
    } else {
        if (QLDS) __syncthreads();
        if (t < t_end) { load_k(t); load_v(t); }
    }
    if (a.window > 0) {                                      // (of this workgroup's rows: the deepest node's window begins last)
#pragma unroll
        for (int r = 0; r < RT; r++) deepest = max(deepest, row_depth[r]);
#pragma unroll
        for (int i = 1; i < 16; i <<= 1) deepest = max(deepest, __shfl_xor(deepest, i, 64));
        if constexpr (RW > 1) {
            __shared__ int depths[RW];
            if (lane == 0) depths[rw] = deepest;
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");    // (the first tiles stay on their way)
#pragma unroll
            for (int i = 0; i < RW; i++) deepest = max(deepest, depths[i]);
        }
        deepest = __builtin_amdgcn_readfirstlane(deepest);
        full_begin = edge + deepest > 0 ? (edge + deepest - 1) / KT + 1 : 0;
    }
    for (; t < t_end; t += KW) {
        const bool more = t + KW < t_end, masked = is_masked(t);
        const char *sk = lds, *sv = lds;
        if constexpr (SHARED) {
            // Tile t has landed when at most the next tile's loads are in flight; behind the barrier everyone's has, and everyone is done with the
            // tile that the next loads overwrite (their LDS reads have returned: the compiler may place the products behind the barrier).  Only of a
            // whole tile it is certain that every wave has issued all its loads.
            if (STAGES == 3 && more && a.D == DP && t + 1 < full_end) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * LOADS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (t + STAGES - 1 < t_end) issue(t + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
            sk = lds + stage * (2 * TILE);
            sv = sk + TILE;
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        }
        if constexpr (SHARED) {
            // 0 * inf: a value that is not finite must not reach the rows that do not see its key, nor what lies behind the last key.  Such values become
            // zeros here; what they do to the rows that see them is put in behind the loop.
            if (masked) {
                const int count = tile_at(t).count;
                T *v = reinterpret_cast<T *>(const_cast<char *>(sv));
                for (int i = tid; i < KT * PIECES; i += 64 * ATTN_WAVES) {
                    const int row = i / PIECES;
                    kvec x = reinterpret_cast<kvec *>(v)[i];
                    bool change = row >= count;
#pragma unroll
                    for (int j = 0; j < U; j++)
                        if (row >= count) x[j] = T(0.f);
                        else if ((bits_of(x[j]) & A::INF) == A::INF) { x[j] = T(0.f); change = true; bad = true; }
                    if (change) reinterpret_cast<kvec *>(v)[i] = x;
                }
                __syncthreads();
            }
            if (idle) continue;
        }
        mvec pf[RT][SPLIT ? 3 : 1];                          // the row tiles' weights as the second product's operand
        f32x4 s[RT][NK];
        if constexpr (SHARED) {
            // (all of K first, V as soon as the scores are under way: no product waits for LDS)
            if constexpr (SPLIT) {
#pragma unroll
                for (int i = 0; i < NK; i++)
#pragma unroll
                    for (int x = 0; x < MS; x++) {
                        const kvec k[2] = {*reinterpret_cast<const kvec *>(sk + piece_at(i * 16 + n16, x * 8 + c * 2)),
                                           *reinterpret_cast<const kvec *>(sk + piece_at(i * 16 + n16, x * 8 + c * 2 + 1))};
                        mvec kp[3];
                        split3<mvec>([&](int j) { return k[j >> 2][j & 3]; }, kp[0], kp[1], kp[2]);
#pragma unroll
                        for (int r = 0; r < RT; r++) s[r][i] = split_mma(kp, qf[r][x], x == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[r][i]);
                    }
            } else {
                kvec kk[NK][KS];
#pragma unroll
                for (int i = 0; i < NK; i++)
#pragma unroll
                    for (int x = 0; x < KS; x++) kk[i][x] = *reinterpret_cast<const kvec *>(sk + piece_at(i * 16 + n16, x * 4 + c));
#pragma unroll
                for (int x = 0; x < KS; x++)
#pragma unroll
                    for (int i = 0; i < NK; i++)
#pragma unroll
                        for (int r = 0; r < RT; r++) s[r][i] = attn_mma<T>(kk[i][x], qf[r][x][0], x == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[r][i]);
                read_v(sv, 0, VL);
            }
        }
#pragma unroll
        for (int r = 0; r < RT; r++) {
            if constexpr (!SHARED) {
#pragma unroll
                for (int i = 0; i < NK; i++) {
                    s[r][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int x = 0; x < KS; x++) {
                        kvec q;
                        if constexpr (QLDS) q = qs[(r * KS + x) * 64 + lane];
                        else q = qf[r][x][0];
                        s[r][i] = attn_mma<T>(kf[i][x], q, s[r][i]);
                    }
                }
            }
            if (masked) {
                const unsigned bits = visible(t, tile_at(t).count, r);
#pragma unroll
                for (int i = 0; i < NK; i++)
#pragma unroll
                    for (int y = 0; y < 4; y++)
                        if (!((bits >> (i * 16 + c * 4 + y)) & 1u)) s[r][i][y] = -INFINITY;
            }
            // online softmax, base 2; the maximum is only raised when it grows by more than LAZY (weights stay below 2^(LAZY + SHIFT))
            float mx = s[r][0][0];
#pragma unroll
            for (int i = 0; i < NK; i++)
#pragma unroll
                for (int y = 0; y < 4; y++) mx = fmaxf(mx, s[r][i][y]);
            mx = max_over_c(mx) * scale2;
            if (__any(mx > m[r] + A::LAZY)) {
                const float mn = fmaxf(m[r], mx), f = mn == m[r] ? 1.f : __builtin_amdgcn_exp2f(m[r] - mn);
                l[r] *= f;
                m[r] = mn;
#pragma unroll
                for (int e = 0; e < E; e++) o[r][e] *= f;
            }
            const float base = (m[r] == -INFINITY ? 0.f : m[r]) - A::SHIFT;
#pragma unroll
            for (int i = 0; i < NK; i++)
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    s[r][i][y] = __builtin_amdgcn_exp2f(fmaf(s[r][i][y], scale2, -base));
                    l[r] += s[r][i][y];
                }
            if constexpr (SPLIT) split3<mvec>([&](int i) { return s[r][i >> 2][i & 3]; }, pf[r][0], pf[r][1], pf[r][2]);
            else
#pragma unroll
                for (int i = 0; i < MU; i++) pf[r][0][i] = from_f32<M>(s[r][i >> 2][i & 3]);
        }
        if constexpr (!SHARED) {
            if (more) load_k(t + KW);
            if (masked) {                                    // (as above)
#pragma unroll
                for (int j = 0; j < VK; j++)
#pragma unroll
                    for (int e = 0; e < E; e++)
                        if ((bits_of(vf[j][e / VU][e % VU]) & A::INF) == A::INF) { vf[j][e / VU][e % VU] = T(0.f); bad = true; }
            }
        }
        // O^T += V^T P^T
#pragma unroll
        for (int e = 0; e < E; e++) {
            if constexpr (SPLIT) {
                if (e % VU == 0) read_v(sv, e / VU, e / VU + 1);
                mvec av[3];
                split3<mvec>([&](int j) { return vf[j][e / VU][e % VU]; }, av[0], av[1], av[2]);
#pragma unroll
                for (int r = 0; r < RT; r++) o[r][e] = split_mma(av, pf[r], o[r][e]);
            } else {
                mvec av;
#pragma unroll
                for (int j = 0; j < VK; j++) av[j] = vf[j][e / VU][e % VU];
#pragma unroll
                for (int r = 0; r < RT; r++) o[r][e] = attn_mma<M>(av, pf[r][0], o[r][e]);
            }
        }
        if constexpr (!SHARED) {
            if (more) load_v(t + KW);
        }
    }
    if (SHARED) bad = __syncthreads_or(bad);
    if (__any(bad) && !idle) {
        // Per masked tile and kind (+inf, -inf, NaN): how many such values a row sees is a product of ones; one makes the sum that kind.
        for (t = t_begin + kw; t < t_end; t += KW) {
            if (!is_masked(t)) continue;
            load_v(t);
#pragma unroll 1
            for (int kind = 0; kind < 3; kind++) {
                const float value = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN;
                const bits_t inf = kind == 0 ? A::INF : (bits_t)(A::INF | A::SIGN);
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    const unsigned sees = visible(t, tile_at(t).count, r);
                    mvec one;
#pragma unroll
                    for (int j = 0; j < VK; j++) one[j] = (sees >> ((j >> 2) * 16 + c * 4 + (j & 3))) & 1u ? M(1.f) : M(0.f);
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        mvec is;
#pragma unroll
                        for (int j = 0; j < VK; j++) {
                            const bits_t x = bits_of(vf[j][e / VU][e % VU]);
                            is[j] = (kind == 2 ? (bits_t)(x & ~A::SIGN) > A::INF : x == inf) ? M(1.f) : M(0.f);
                        }
                        const f32x4 n = attn_mma<M>(is, one, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                        for (int y = 0; y < 4; y++)
                            if (n[y] > 0.f) o[r][e][y] += value;
                    }
                }
            }
        }
    }
    __syncthreads();

    // join the key waves: common maximum, then the outputs one wave after another (a fixed order)
#pragma unroll
    for (int r = 0; r < RT; r++) {
        l[r] = sum_over_c(l[r]);
        if (c == 0) { sm[kw * ROWS + rw * WROWS + r * 16 + n16] = m[r]; sl[kw * ROWS + rw * WROWS + r * 16 + n16] = l[r]; }
    }
    __syncthreads();
    if constexpr (KW > 1) {
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const int row = rw * WROWS + r * 16 + n16;
            float mm = sm[row];
#pragma unroll
            for (int w = 1; w < KW; w++) mm = fmaxf(mm, sm[w * ROWS + row]);
            const float f = m[r] == mm ? 1.f : __builtin_amdgcn_exp2f(m[r] - mm);
#pragma unroll
            for (int e = 0; e < E; e++) o[r][e] *= f;
        }
    }
#pragma unroll
    for (int w = 0; w < KW; w++) {
        if (w == kw) {
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int y = 0; y < 4; y++)
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        f32x4 *dst = reinterpret_cast<f32x4 *>(&so[(rw * WROWS + r * 16 + n16) * LD + ((e / VU) * 16 + c * 4 + y) * VU + e % VU]);
                        const f32x4 x = {o[r][e][y], o[r][e + 1][y], o[r][e + 2][y], o[r][e + 3][y]};
                        *dst = w == 0 ? x : *dst + x;
                    }
        }
        __syncthreads();
    }
    const bool whole = tr.per >= tr.n_all;                   // one split holds all keys of this sequence
    const int64_t prow = ((int64_t)split * gridDim.y + b) * a.Hk + kvh;
    for (int row = wave; row < ROWS && row0 + row < R; row += ATTN_WAVES) {
        float mm = sm[row], total = 0.f;
#pragma unroll
        for (int w = 1; w < KW; w++) mm = fmaxf(mm, sm[w * ROWS + row]);
#pragma unroll
        for (int w = 0; w < KW; w++) total += sl[w * ROWS + row] * (sm[w * ROWS + row] == mm ? 1.f : __builtin_amdgcn_exp2f(sm[w * ROWS + row] - mm));
        const int grow = row0 + row, node = grow / a.G, h = kvh * a.G + (grow - node * a.G);
        if (whole) {
            const bool none = total == 0.f || a.depth[(size_t)b * a.T + node] < 0;
            T *out = (T *)a.out + b * a.o_sb + node * a.o_st + h * a.o_sh;
            for (int d = lane; d < a.D; d += 64) out[d] = from_f32<T>(none ? 0.f : so[row * LD + d] / total);
            if (a.lse && lane == 0) a.lse[((size_t)b * a.T + node) * a.H + h] = none ? -INFINITY : (mm - A::SHIFT + log2f(total)) * 0.693147180559945309417f;
        } else {
            for (int d = lane; d < a.D; d += 64) plan.part_o[(prow * R + grow) * a.D + d] = so[row * LD + d];
            if (lane == 0) { plan.part_ml[(prow * R + grow) * 2] = mm; plan.part_ml[(prow * R + grow) * 2 + 1] = total; }
        }
    }
}

// Joins the parts of a row: one wave per (row, kv head, sequence); grid (ceil(rows / 4), Hk, batch).  L lanes take one part's outputs, four values
// each (the matrix-pipe form's head_dim is a multiple of four), 64 / L parts at a time, their weights first: bound by the read of the parts.
template <typename T, int L, bool SHARED> __global__ __launch_bounds__(256) void k_tree_attn_join(TreeAttnArgs a, TreeAttnPlan plan) {
    typedef AttnType<T> A;
    const int lane = threadIdx.x & 63, R = a.T * a.G, row = blockIdx.x * 4 + (threadIdx.x >> 6), kvh = blockIdx.y, b = blockIdx.z;
    if (row >= R) return;
    const TileRange tr = tile_range<ATTN_KT<T, SHARED>>(a, b, plan.splits, SHARED ? 1 : ATTN_WAVES);
    const int n = (tr.n_all + tr.per - 1) / tr.per;          // at most 64 parts: lane s holds part s's weight
    if (n <= 1) return;                                      // written by its only part
    const int64_t step = (int64_t)gridDim.z * a.Hk * R, at = ((int64_t)b * a.Hk + kvh) * R + row;
    const float ms = lane < n ? plan.part_ml[(lane * step + at) * 2] : -INFINITY, ls = lane < n ? plan.part_ml[(lane * step + at) * 2 + 1] : 0.f;
    const float mm = wave_max(ms), f = ms == mm ? 1.f : __builtin_amdgcn_exp2f(ms - mm);
    const float total = wave_sum(f * ls);
    const int g = lane / L, d = (lane % L) * 4;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < n; s += 64 / L) {
        const float w = __shfl(f, s + g, 64);
        if (s + g < n && d < a.D) acc += w * *reinterpret_cast<const f32x4 *>(plan.part_o + ((s + g) * step + at) * a.D + d);
    }
#pragma unroll
    for (int o = L; o < 64; o <<= 1)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] += __shfl_xor(acc[i], o, 64);
    const int node = row / a.G, h = kvh * a.G + (row - node * a.G);
    const bool none = total == 0.f || a.depth[(size_t)b * a.T + node] < 0;
    if (g == 0 && d < a.D) {
        T *out = (T *)a.out + b * a.o_sb + node * a.o_st + h * a.o_sh + d;
#pragma unroll
        for (int i = 0; i < 4; i++) out[i] = from_f32<T>(none ? 0.f : acc[i] / total);
    }
    if (a.lse && lane == 0) a.lse[((size_t)b * a.T + node) * a.H + h] = none ? -INFINITY : (mm - A::SHIFT + log2f(total)) * 0.693147180559945309417f;
}

}  // namespace vox
