// vox_ops.hip — the C entries of include/vox_hip_ops.h: checks on the host, then the launches.  The kernels are in the headers below.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>
#include <algorithm>
#include <atomic>

#include "../../include/vox_hip_ops.h"
#include "vox_ops_common.h"
#include "vox_tree.h"
#include "vox_tree_attn.h"
#include "vox_token_scores.h"
#include "vox_linear_i8.h"

using namespace vox;

__attribute__((visibility("hidden"))) void vox_set_last_error(const char *text);      // vox_hip_engine.hip: what vox_hip_last_error() gives

namespace {

int refuse(const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    vox_set_last_error(buf);
    return -1;
}
#define CHECK(cond, ...) do { if (!(cond)) return refuse(__VA_ARGS__); } while (0)

// The caller's current device is put back when the call ends.  Only gfx950: the code object holds nothing else.
struct OnDevice {
    int before = -1, device;
    bool ok = false;
    OnDevice(const char *who, int dev) : device(dev) {
        static std::atomic<int> known[64];                   // 0 not asked, 1 gfx950, 2 something else
        if (dev < 0 || dev >= 64 || hipGetDevice(&before) != hipSuccess) { (void)hipGetLastError(); refuse("%s: no such device (%d)", who, dev); return; }
        int k = known[dev].load(std::memory_order_relaxed);
        if (k == 0) {
            hipDeviceProp_t prop;
            if (hipGetDeviceProperties(&prop, dev) != hipSuccess) { (void)hipGetLastError(); refuse("%s: no such device (%d)", who, dev); return; }
            k = strncmp(prop.gcnArchName, "gfx950", 6) == 0 ? 1 : 2;
            known[dev].store(k, std::memory_order_relaxed);
        }
        if (k != 1) { refuse("%s: device %d is not gfx950: these kernels are written for MI355X only", who, dev); return; }
        if (before != dev && hipSetDevice(dev) != hipSuccess) { (void)hipGetLastError(); refuse("%s: hipSetDevice(%d) failed", who, dev); return; }
        (void)hipGetLastError();                             // an earlier call's error is not this launch's (launched() asks the thread's last one)
        ok = true;
    }
    ~OnDevice() { if (ok && before != device) (void)hipSetDevice(before); }
};

int launched(const char *who) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : refuse("%s: launch failed: %s", who, hipGetErrorString(e));
}

constexpr int64_t GRID_MAX = ((int64_t)1 << 24) - 1;         // workgroups of 256 along a grid's first dimension (its threads are counted in 32 bits)
int dtype_size(int dtype) { return dtype == VOX_F32 ? 4 : dtype == VOX_BF16 || dtype == VOX_F16 ? 2 : 0; }
bool aligned(const void *p, int64_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
// One call of f with the element type as a template argument.
template <typename F> void by_type(int dtype, F f) {
    if (dtype == VOX_F32) f(float{});
    else if (dtype == VOX_BF16) f(bf16_t{});
    else f(f16_t{});
}

}  // namespace

// ---- draft trees -------------------------------------------------------------------------------------------------------------
extern "C" int vox_hip_tree_plan(const int32_t *parents, const int32_t *n_nodes, int batch, int nodes, uint64_t *ancestors, int32_t *depth,
                                 int device, void *stream) {
    CHECK(batch >= 0 && batch <= GRID_MAX && nodes >= 0 && nodes <= VOX_TREE_MAX_NODES, "vox_hip_tree_plan: batch %d, nodes %d (at most %d nodes)", batch, nodes, VOX_TREE_MAX_NODES);
    if (batch == 0 || nodes == 0) return 0;
    CHECK(parents && ancestors && depth, "vox_hip_tree_plan: null pointer");
    OnDevice on("vox_hip_tree_plan", device);
    if (!on.ok) return -1;
    hipLaunchKernelGGL(k_tree_plan, dim3(batch), dim3(TREE_MAX), 0, (hipStream_t)stream, parents, n_nodes, nodes, ancestors, depth);
    return launched("vox_hip_tree_plan");
}

extern "C" int vox_hip_tree_accept(const int32_t *tokens, const int32_t *choices, const int32_t *root_choice, const int32_t *parents,
                                   const uint64_t *ancestors, const int32_t *depth, const int32_t *cache_len, int batch, int nodes, int32_t *path,
                                   int32_t *n_accepted, int32_t *next_token, int32_t *new_len, int device, void *stream) {
    CHECK(batch >= 0 && batch <= GRID_MAX && nodes >= 1 && nodes <= VOX_TREE_MAX_NODES, "vox_hip_tree_accept: batch %d, nodes %d (1 to %d nodes)", batch, nodes, VOX_TREE_MAX_NODES);
    if (batch == 0) return 0;
    CHECK(tokens && choices && root_choice && parents && ancestors && depth && cache_len && path && n_accepted && next_token && new_len,
          "vox_hip_tree_accept: null pointer");
    OnDevice on("vox_hip_tree_accept", device);
    if (!on.ok) return -1;
    hipLaunchKernelGGL(k_tree_accept, dim3(batch), dim3(TREE_MAX), 0, (hipStream_t)stream, tokens, choices, root_choice, parents, ancestors, depth,
                       cache_len, nodes, path, n_accepted, next_token, new_len);
    return launched("vox_hip_tree_accept");
}

extern "C" int vox_hip_tree_commit(int dtype, int layers, int batch, int nodes, int kv_heads, int head_dim, int cap, const void *k,
                                   const int64_t *k_strides, const void *v, const int64_t *v_strides, void *k_cache, const int64_t *kc_strides,
                                   void *v_cache, const int64_t *vc_strides, const int32_t *path, const int32_t *n_accepted, const int32_t *cache_len,
                                   int device, void *stream) {
    const int size = dtype_size(dtype);
    CHECK(size, "vox_hip_tree_commit: dtype %d", dtype);
    CHECK(layers >= 0 && layers <= 32767 && batch >= 0 && batch <= GRID_MAX && nodes >= 0 && nodes <= VOX_TREE_MAX_NODES && kv_heads >= 1 && kv_heads <= 4096 && head_dim >= 1 && head_dim <= 4096,
          "vox_hip_tree_commit: layers %d, batch %d, nodes %d, kv_heads %d, head_dim %d", layers, batch, nodes, kv_heads, head_dim);
    if (layers == 0 || batch == 0 || nodes == 0) return 0;
    CHECK(cap >= nodes, "vox_hip_tree_commit: a ring of %d rows does not hold a path of %d nodes", cap, nodes);
    CHECK(k && v && k_cache && v_cache && k_strides && v_strides && kc_strides && vc_strides && path && n_accepted && cache_len, "vox_hip_tree_commit: null pointer");
    TreeCommitArgs a{(const char *)k, (const char *)v, (char *)k_cache, (char *)v_cache, {}, {}, {}, {}, path, n_accepted, cache_len, nodes, kv_heads, head_dim * size, cap};
    uint64_t all = (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_cache | (uintptr_t)v_cache | (uint64_t)a.head_bytes | 16;
    for (int i = 0; i < 4; i++) {
        CHECK(k_strides[i] >= 0 && v_strides[i] >= 0 && kc_strides[i] >= 0 && vc_strides[i] >= 0, "vox_hip_tree_commit: negative stride");
        a.k_s[i] = k_strides[i] * size; a.v_s[i] = v_strides[i] * size; a.kc_s[i] = kc_strides[i] * size; a.vc_s[i] = vc_strides[i] * size;
        all |= a.k_s[i] | a.v_s[i] | a.kc_s[i] | a.vc_s[i];
    }
    OnDevice on("vox_hip_tree_commit", device);
    if (!on.ok) return -1;
    const dim3 grid(batch, layers * 2, (nodes + COMMIT_ROWS - 1) / COMMIT_ROWS);
    switch (all & -all) {                                    // the widest access that every address allows
        case 16: hipLaunchKernelGGL(k_tree_commit<uint4>, grid, dim3(256), 0, (hipStream_t)stream, a); break;
        case 8: hipLaunchKernelGGL(k_tree_commit<uint2>, grid, dim3(256), 0, (hipStream_t)stream, a); break;
        case 4: hipLaunchKernelGGL(k_tree_commit<uint32_t>, grid, dim3(256), 0, (hipStream_t)stream, a); break;
        case 2: hipLaunchKernelGGL(k_tree_commit<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, a); break;
        default: return refuse("vox_hip_tree_commit: pointers are not aligned to their elements");
    }
    return launched("vox_hip_tree_commit");
}

// ---- attention ---------------------------------------------------------------------------------------------------------------
namespace {
int check_attn(const vox_hip_tree_attn_t *a) {
    const char *who = "vox_hip_tree_attention";
    CHECK(a, "%s: null arguments", who);
    CHECK(dtype_size(a->dtype), "%s: dtype %d", who, a->dtype);
    CHECK(a->batch >= 0 && a->batch <= 65535, "%s: batch %d (at most 65535)", who, a->batch);
    CHECK(a->nodes >= 0 && a->nodes <= VOX_TREE_MAX_NODES, "%s: %d nodes (at most %d)", who, a->nodes, VOX_TREE_MAX_NODES);
    CHECK(a->kv_heads >= 1 && a->heads >= 1 && a->heads <= 4096 && a->heads % a->kv_heads == 0, "%s: %d heads over %d kv heads", who, a->heads, a->kv_heads);
    CHECK(a->head_dim >= 1 && a->head_dim <= TREE_SCALAR_MAX_D, "%s: head_dim %d (at most %d)", who, a->head_dim, TREE_SCALAR_MAX_D);
    CHECK(a->cap >= 1, "%s: a cache of %d rows", who, a->cap);
    CHECK(a->scale != 0.f && a->scale >= -2e38f && a->scale <= 2e38f, "%s: scale %g (a finite number other than 0, of at most 2e38)", who, (double)a->scale);      // (times log2 e)
    CHECK(a->reserved == 0, "%s: reserved is not 0", who);
    return 0;
}

// The matrix-pipe kernel takes 16-byte loads: every row of every operand starts on 16 bytes and holds whole loads, and keys lie less than 2^26
// bytes apart (offsets within a tile are 32 bits).  Everything else runs on the scalar kernel.
bool attn_wide(const vox_hip_tree_attn_t *a) {
    const int size = dtype_size(a->dtype), unit = 16 / size;
    const void *p[5] = {a->q, a->k, a->v, a->k_cache, a->v_cache};
    for (const void *x : p)
        if (!aligned(x, 16)) return false;
    const int64_t *st = &a->q_sb;
    for (int i = 0; i < 15; i++)
        if (st[i] % unit) return false;
    const int64_t rows[4] = {a->k_st, a->v_st, a->kc_ss, a->vc_ss};
    for (int64_t r : rows)
        if (r * size >= (int64_t)1 << 26) return false;
    return a->head_dim % unit == 0;
}
// Up to 16 rows (nodes x heads of a kv head; 32 where a head has up to 64 dimensions) the waves of a workgroup have keys of their own, above that
// rows of their own (64 or 128 per workgroup) and shared keys.  32 rows of 128 dimensions over 4 x 16000 keys: own 78 us, shared 57 in bf16; 152 and 125
// in f32.  64 dimensions, 4 x 16000 keys, own / shared: f32 32 rows 58 / 73 us, 36 rows 91 / 74; bf16 32 rows 36 / 33, 36 rows 45 / 34; over 8 x 1000 keys
// the two are within 10 % of each other.  Splits: enough workgroups for two per CU, but at least one key tile per wave in each.
struct AttnLaunch { bool wide, shared; int DP, RT, row_blocks, key_waves, splits; int64_t ws; };
AttnLaunch attn_launch(const vox_hip_tree_attn_t *a) {
    AttnLaunch l{};
    l.wide = attn_wide(a);
    if (!l.wide || a->batch == 0 || a->nodes == 0) return l;
    const int64_t R = (int64_t)a->nodes * (a->heads / a->kv_heads);
    l.DP = a->head_dim <= 64 ? 64 : a->head_dim <= 128 ? 128 : 256;
    l.shared = R > (l.DP > 64 ? 16 : 32);
    l.RT = l.DP == 256 || R <= 16 || (l.shared && R <= 64) ? 1 : 2;
    const int rows = l.RT * 16 * (l.shared ? ATTN_WAVES : 1);
    l.key_waves = l.shared ? 1 : ATTN_WAVES;
    l.row_blocks = (int)((R + rows - 1) / rows);
    const int KT = a->dtype == VOX_F32 && !l.shared ? 16 : 32;
    const int64_t keys = a->window > 0 ? std::min(a->cap, a->window) : a->cap, tiles = (keys + KT - 1) / KT + (a->nodes + KT - 1) / KT;
    const int64_t groups = (int64_t)a->batch * a->kv_heads * l.row_blocks;
    l.splits = (int)std::max<int64_t>(1, std::min<int64_t>({64, 512 / groups, (tiles + l.key_waves - 1) / l.key_waves}));
    if (l.splits > 1) l.ws = round_up((int64_t)l.splits * a->batch * a->kv_heads * R * a->head_dim * 4, 256) + (int64_t)l.splits * a->batch * a->kv_heads * R * 8;
    return l;
}
template <typename T, int DP, int RT, bool SHARED> void launch_attn2(const TreeAttnArgs &t, const TreeAttnPlan &p, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((k_tree_attn<T, DP, RT, SHARED>), grid, dim3(64 * ATTN_WAVES), (attn_lds<T, DP, RT, SHARED>()), s, t, p);
}
template <typename T, bool SHARED> void launch_attn_join(const TreeAttnArgs &t, const TreeAttnPlan &p, int DP, int batch, hipStream_t s) {
    const dim3 grid((t.T * t.G + 3) / 4, t.Hk, batch);
    if (DP == 64) hipLaunchKernelGGL((k_tree_attn_join<T, 16, SHARED>), grid, dim3(256), 0, s, t, p);
    else if (DP == 128) hipLaunchKernelGGL((k_tree_attn_join<T, 32, SHARED>), grid, dim3(256), 0, s, t, p);
    else hipLaunchKernelGGL((k_tree_attn_join<T, 64, SHARED>), grid, dim3(256), 0, s, t, p);
}
template <typename T, int DP> void launch_attn(const TreeAttnArgs &t, const TreeAttnPlan &p, const AttnLaunch &l, dim3 grid, hipStream_t s) {
    if constexpr (DP == 256) {
        if (l.shared) launch_attn2<T, DP, 1, true>(t, p, grid, s);
        else launch_attn2<T, DP, 1, false>(t, p, grid, s);
    } else {
        if (l.shared && l.RT == 2) launch_attn2<T, DP, 2, true>(t, p, grid, s);
        else if (l.shared) launch_attn2<T, DP, 1, true>(t, p, grid, s);
        else if (l.RT == 1) launch_attn2<T, DP, 1, false>(t, p, grid, s);
        else if constexpr (DP == 64) launch_attn2<T, DP, 2, false>(t, p, grid, s);
    }
}
}  // namespace
extern "C" int64_t vox_hip_tree_attention_workspace(const vox_hip_tree_attn_t *a) {
    if (check_attn(a)) return -1;
    return attn_launch(a).ws;
}
extern "C" int vox_hip_tree_attention(const vox_hip_tree_attn_t *a, void *ws, size_t ws_bytes, int device, void *stream) {
    if (check_attn(a)) return -1;
    if (a->batch == 0 || a->nodes == 0) return 0;
    CHECK(a->q && a->k && a->v && a->k_cache && a->v_cache && a->cache_len && a->ancestors && a->depth && a->out, "vox_hip_tree_attention: null pointer");
    const int64_t *st = &a->q_sb;
    for (int i = 0; i < 18; i++) CHECK(st[i] >= 0, "vox_hip_tree_attention: negative stride");
    const AttnLaunch l = attn_launch(a);
    CHECK(l.ws == 0 || (ws && aligned(ws, 256) && ws_bytes >= (size_t)l.ws), "vox_hip_tree_attention: needs %lld bytes of workspace, 256-byte aligned", (long long)l.ws);
    OnDevice on("vox_hip_tree_attention", device);
    if (!on.ok) return -1;
    TreeAttnArgs t{a->q, a->k, a->v, a->k_cache, a->v_cache, a->cache_len, a->ancestors, a->depth, a->out, a->lse,
                   a->q_sb, a->q_st, a->q_sh, a->k_sb, a->k_st, a->k_sh, a->v_sb, a->v_st, a->v_sh, a->kc_sb, a->kc_ss, a->kc_sh, a->vc_sb, a->vc_ss, a->vc_sh,
                   a->o_sb, a->o_st, a->o_sh, a->nodes, a->heads, a->kv_heads, a->heads / a->kv_heads, a->head_dim, a->cap, a->window, (a->nodes + 63) / 64, a->scale};
    const hipStream_t s = (hipStream_t)stream;
    if (!l.wide) {
        by_type(a->dtype, [&](auto z) {
            hipLaunchKernelGGL(k_tree_attn_scalar<decltype(z)>, dim3(a->nodes * a->heads, a->batch), dim3(256), 0, s, t);
        });
        return launched("vox_hip_tree_attention");
    }
    const int R = a->nodes * t.G;
    TreeAttnPlan p{l.splits, l.row_blocks, (float *)ws, (float *)((char *)ws + round_up((int64_t)l.splits * a->batch * a->kv_heads * R * a->head_dim * 4, 256))};
    const dim3 grid((unsigned)(round_up((int64_t)l.splits * a->kv_heads, 8) * l.row_blocks), a->batch);
    by_type(a->dtype, [&](auto z) {
        typedef decltype(z) T;
        if (l.DP == 64) launch_attn<T, 64>(t, p, l, grid, s);
        else if (l.DP == 128) launch_attn<T, 128>(t, p, l, grid, s);
        else launch_attn<T, 256>(t, p, l, grid, s);
        if (l.splits > 1 && l.shared) launch_attn_join<T, true>(t, p, l.DP, a->batch, s);
        else if (l.splits > 1) launch_attn_join<T, false>(t, p, l.DP, a->batch, s);
    });
    return launched("vox_hip_tree_attention");
}

// ---- token scores ------------------------------------------------------------------------------------------------------------
namespace {
struct ScorePlan { int parts, part_len; int64_t ws; };
ScorePlan score_plan(int64_t rows, int vocab, int top) {
    // Rows are cut until there are about four workgroups per CU, parts down to one trip of a workgroup (SC_UNROLL loads of 16 bytes per thread): a
    // row of 131072 on its own takes 32 workgroups and 13 us with the join; 386 rows take three each.
    const int step = SC_THREADS * 8, trip = SC_THREADS * SC_UNROLL * 4;
    const int parts = (int)std::max<int64_t>(1, std::min<int64_t>({SC_MAX_PARTS, (1024 + rows / 2) / std::max<int64_t>(rows, 1), vocab / trip}));
    ScorePlan p;
    p.part_len = (int)round_up((vocab + parts - 1) / parts, step);
    p.parts = (vocab + p.part_len - 1) / p.part_len;
    p.ws = p.parts == 1 ? 0 : round_up(rows * p.parts * (int64_t)sizeof(RowSum), 256) + rows * p.parts * top * 8;
    return p;
}
int check_scores(int dtype, int64_t rows, int vocab, int top) {
    CHECK(dtype_size(dtype), "vox_hip_token_scores: dtype %d", dtype);
    CHECK(rows >= 0 && rows <= GRID_MAX, "vox_hip_token_scores: %lld rows (at most %lld)", (long long)rows, (long long)GRID_MAX);
    CHECK(vocab >= 1 && vocab <= (1 << 30), "vox_hip_token_scores: a vocabulary of %d", vocab);
    CHECK(top >= 0 && top <= VOX_SCORES_MAX_TOP && top <= vocab, "vox_hip_token_scores: top %d of %d (at most %d)", top, vocab, VOX_SCORES_MAX_TOP);
    return 0;
}
}  // namespace
extern "C" int64_t vox_hip_token_scores_workspace(int dtype, int64_t rows, int vocab, int top) {
    return check_scores(dtype, rows, vocab, top) ? -1 : score_plan(rows, vocab, top).ws;
}
extern "C" int vox_hip_token_scores(int dtype, const void *logits, int64_t row_stride, int64_t rows, int vocab, const int32_t *tokens, int given, int top,
                                    float *logprob, float *entropy, float *lse, int32_t *top_index, float *top_logprob, void *ws, size_t ws_bytes,
                                    int device, void *stream) {
    if (check_scores(dtype, rows, vocab, top)) return -1;
    CHECK(given >= 0 && given <= (1 << 20), "vox_hip_token_scores: %d given tokens", given);
    CHECK(row_stride >= 0, "vox_hip_token_scores: negative stride");
    if (rows == 0) return 0;
    CHECK(logits && entropy && lse && (given == 0 || (tokens && logprob)) && (top == 0 || (top_index && top_logprob)), "vox_hip_token_scores: null pointer");
    const ScorePlan p = score_plan(rows, vocab, top);
    CHECK(p.ws == 0 || (ws && aligned(ws, 256) && ws_bytes >= (size_t)p.ws), "vox_hip_token_scores: needs %lld bytes of workspace, 256-byte aligned", (long long)p.ws);
    OnDevice on("vox_hip_token_scores", device);
    if (!on.ok) return -1;
    const int size = dtype_size(dtype);
    ScoreArgs a{logits, row_stride, vocab, given, top, p.parts, p.part_len, tokens, logprob, entropy, lse, top_index, top_logprob, (RowSum *)ws,
                (uint64_t *)((char *)ws + round_up(rows * p.parts * (int64_t)sizeof(RowSum), 256))};
    const bool wide = aligned(logits, 16) && row_stride * size % 16 == 0;
    const dim3 grid((unsigned)(rows * p.parts));
    by_type(dtype, [&](auto z) {
        typedef decltype(z) T;
        if (wide) hipLaunchKernelGGL((k_token_scores<T, 16 / sizeof(T)>), grid, dim3(SC_THREADS), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((k_token_scores<T, 1>), grid, dim3(SC_THREADS), 0, (hipStream_t)stream, a);
        if (p.parts > 1) hipLaunchKernelGGL(k_token_scores_join<T>, dim3((unsigned)rows), dim3(SC_THREADS), 0, (hipStream_t)stream, a);
    });
    return launched("vox_hip_token_scores");
}

// ---- 8-bit integers ----------------------------------------------------------------------------------------------------------
namespace {
constexpr int I8_MAX_ROWS = 65535 * 64;                      // (a grid's second dimension; and 2^32 threads of the quantiser's)
int check_i8(const char *who, int dtype, int64_t rows, int K) {
    CHECK(dtype_size(dtype), "%s: dtype %d", who, dtype);
    CHECK(rows >= 0 && rows <= I8_MAX_ROWS, "%s: %lld rows (at most %d)", who, (long long)rows, I8_MAX_ROWS);
    CHECK(K >= 1 && K <= VOX_I8_MAX_K, "%s: K %d (1 to %d)", who, K, VOX_I8_MAX_K);
    return 0;
}
int i8_ldq(int K) { return (int)round_up(K, I8_BK); }
template <typename T> void launch_quant(const T *x, int64_t stride, int64_t rows, int K, int ldq, int8_t *q, float *scale, hipStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const bool wide = K % N == 0 && ldq % N == 0 && stride % N == 0 && aligned(x, 16) && aligned(q, 8);
    const int threads = (int)std::min<int64_t>(round_up((ldq + (wide ? N : 1) - 1) / (wide ? N : 1), 64), I8_QUANT_THREADS);      // one load per thread where that is enough
    if (wide) hipLaunchKernelGGL((k_quant_rows_i8<T, N>), dim3((unsigned)rows), dim3(threads), 0, s, x, stride, K, ldq, q, scale);
    else hipLaunchKernelGGL((k_quant_rows_i8<T, 1>), dim3((unsigned)rows), dim3(threads), 0, s, x, stride, K, ldq, q, scale);
}
// Up to 32 rows the product is a read of the weights (k_linear_i8_rows).  Above, tiles of 128 rows x 128 channels, of 64 rows where there would be
// fewer than 192; K is split where even those are fewer than 100, into parts of six slices of 128 or more: the parts' way through memory and
// the third launch cost 6 - 9 us.  Whole / split: K 5120, 10 tiles 24.3 / 16.2 us, 40 tiles 25.3 / 18.7, 80 tiles 25.7 / 20.8, 120 tiles 27.3 / 24.3 (the limit
// leaves these whole), 160 tiles 28.7 / 31.7; K 2560, 80 tiles 16.9 / 18.7 (and splits these).
struct I8Plan { bool few; int BM, tiles_m, tiles_n, splits; int64_t scale_at, part_at, ws; };
I8Plan i8_plan(int64_t rows, int K, int N, bool wide) {
    I8Plan p{};
    p.splits = 1;
    p.few = wide && rows <= I8_FEW_ROWS && rows * K <= I8_FEW;
    if (p.few) return p;
    p.scale_at = round_up(rows * i8_ldq(K), 256);
    p.part_at = p.ws = p.scale_at + round_up(rows * 4, 256);
    if (!wide || rows <= 32 || N == 0) return p;
    p.tiles_n = (N + I8_BN - 1) / I8_BN;
    for (p.BM = 128;; p.BM = 64) {
        p.tiles_m = (int)((rows + p.BM - 1) / p.BM);
        if (p.BM == 64 || (int64_t)p.tiles_m * p.tiles_n >= 192) break;
    }
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    if (tiles < 100) p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(256 / tiles, i8_ldq(K) / I8_BK / 6));
    if (p.splits > 1) p.ws += (int64_t)p.splits * p.tiles_m * p.BM * p.tiles_n * I8_BN * 4;
    return p;
}
template <typename T, int BM, int STAGES> void launch_i8_tile(const LinearI8Args &a, const I8Plan &p, hipStream_t s) {
    const int64_t total = (int64_t)p.tiles_m * p.tiles_n * p.splits;
    hipLaunchKernelGGL((k_linear_i8_tile<T, BM, STAGES>), dim3((unsigned)round_up(total, 8)), dim3(256), (i8_tile_lds<T, BM, STAGES>()), s, a, p.tiles_m, p.tiles_n);
    if (p.splits > 1) {
        const int64_t ld = (int64_t)p.tiles_n * I8_BN, groups = (int64_t)a.M * ((a.N + 3) / 4);
        hipLaunchKernelGGL(k_linear_i8_join<T>, dim3((unsigned)std::min<int64_t>((groups + 255) / 256, 2048)), dim3(256), 0, s, a, ld, ld * p.tiles_m * BM);
    }
}
}  // namespace
extern "C" int vox_hip_quantize_rows_i8(int dtype, const void *x, int64_t row_stride, int64_t rows, int K, int8_t *q, float *scale, int device, void *stream) {
    if (check_i8("vox_hip_quantize_rows_i8", dtype, rows, K)) return -1;
    CHECK(row_stride >= 0, "vox_hip_quantize_rows_i8: negative stride");
    if (rows == 0) return 0;
    CHECK(x && q && scale, "vox_hip_quantize_rows_i8: null pointer");
    OnDevice on("vox_hip_quantize_rows_i8", device);
    if (!on.ok) return -1;
    by_type(dtype, [&](auto z) {
        typedef decltype(z) T;
        launch_quant<T>((const T *)x, row_stride, rows, K, K, q, scale, (hipStream_t)stream);
    });
    return launched("vox_hip_quantize_rows_i8");
}
namespace {
bool i8_wide(int K, const int8_t *w, int64_t w_stride) { return K % 16 == 0 && w_stride % 16 == 0 && aligned(w, 16); }
}  // namespace
extern "C" int64_t vox_hip_linear_i8_workspace(int dtype, int64_t rows, int K, int N, const int8_t *w, int64_t w_stride) {
    if (check_i8("vox_hip_linear_i8", dtype, rows, K)) return -1;
    CHECK(N >= 0 && N <= (1 << 24) && (rows / 64 + 1) * (N / 128 + 1) <= GRID_MAX / 8, "vox_hip_linear_i8: N %d, %lld rows", N, (long long)rows);
    return i8_plan(rows, K, N, i8_wide(K, w, w_stride)).ws;
}
extern "C" int vox_hip_linear_i8(int dtype, const void *x, int64_t x_stride, int64_t rows, int K, int N, const int8_t *w, int64_t w_stride, const float *w_scale,
                                 const void *bias, void *y, int64_t y_stride, void *ws, size_t ws_bytes, int device, void *stream) {
    const int64_t need = vox_hip_linear_i8_workspace(dtype, rows, K, N, w, w_stride);
    if (need < 0) return -1;
    CHECK(x_stride >= 0 && w_stride >= 0 && (y_stride >= N || rows <= 1), "vox_hip_linear_i8: strides %lld, %lld, %lld", (long long)x_stride, (long long)w_stride, (long long)y_stride);
    if (rows == 0 || N == 0) return 0;
    CHECK(x && w && w_scale && y, "vox_hip_linear_i8: null pointer");
    CHECK(need == 0 || (ws && aligned(ws, 256) && ws_bytes >= (size_t)need), "vox_hip_linear_i8: needs %lld bytes of workspace, 256-byte aligned", (long long)need);
    OnDevice on("vox_hip_linear_i8", device);
    if (!on.ok) return -1;
    const int ldq = i8_ldq(K);
    int8_t *xq = (int8_t *)ws;
    const bool wide = i8_wide(K, w, w_stride);
    const I8Plan p = i8_plan(rows, K, N, wide);
    float *xs = (float *)((char *)ws + p.scale_at);
    LinearI8Args a{xq, xs, w, w_stride, w_scale, bias, y, y_stride, (int)rows, K, N, ldq, (int *)((char *)ws + p.part_at), p.splits};
    const hipStream_t st = (hipStream_t)stream;
    by_type(dtype, [&](auto z) {
        typedef decltype(z) T;
        if (p.few) {
            constexpr int V = 16 / sizeof(T);
            const unsigned lds = (unsigned)(rows * (ldq + 16));
            if (K % V == 0 && x_stride % V == 0 && aligned(x, 16)) hipLaunchKernelGGL((k_linear_i8_few<T, V>), dim3((N + 15) / 16), dim3(64 * I8_ROWS_WAVES), lds, st, a, (const T *)x, x_stride);
            else hipLaunchKernelGGL((k_linear_i8_few<T, 1>), dim3((N + 15) / 16), dim3(64 * I8_ROWS_WAVES), lds, st, a, (const T *)x, x_stride);
            return;
        }
        launch_quant<T>((const T *)x, x_stride, rows, K, ldq, xq, xs, st);
        const dim3 narrow((N + 15) / 16);
        if (!wide) hipLaunchKernelGGL(k_linear_i8_bytes<T>, dim3((N + 63) / 64, (unsigned)((rows + 63) / 64)), dim3(256), 0, st, a);
        else if (rows <= 16) hipLaunchKernelGGL((k_linear_i8_rows<T, 1>), narrow, dim3(64 * I8_ROWS_WAVES), 0, st, a);
        else if (rows <= 32) hipLaunchKernelGGL((k_linear_i8_rows<T, 2>), narrow, dim3(64 * I8_ROWS_WAVES), 0, st, a);
        else if (p.BM == 128) launch_i8_tile<T, 128, 2>(a, p, st);
        else launch_i8_tile<T, 64, 3>(a, p, st);
    });
    return launched("vox_hip_linear_i8");
}
