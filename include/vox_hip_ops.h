/*
 * vox_hip_ops.h — operators on device memory for a draft-verification step (libvoxhip.so, gfx950 only).
 *
 * A verification pass takes several drafted tokens through the decoder at once.  The drafts form a tree: node i of a sequence
 * has a parent among the earlier nodes, or -1 for the end of the cache; a node sits at position cache_len + depth.  Per pass:
 *   vox_hip_tree_plan        parents -> ancestor sets and depths (once per pass, all layers use them)
 *   vox_hip_linear_i8        the nodes' rows through a matrix of 8-bit integers
 *   vox_hip_tree_attention   the nodes' queries over the ring cache and their own ancestors (once per layer)
 *   vox_hip_token_scores     rows of logits -> log probabilities of given tokens, entropy, top alternatives
 *   vox_hip_tree_accept      drafts that agree with the model's choices -> accepted path, next token, new length
 *   vox_hip_tree_commit      the path's keys and values into the ring cache (all layers in one launch)
 *
 * Conventions: every pointer is device memory of `device` unless its comment says host; `stream` is a hipStream_t of that
 * device (NULL = its null stream; vox_hip_stream_handle gives an engine's).  The calls enqueue and return; nothing waits.  They keep
 * no state and allocate nothing: scratch memory is the caller's (`ws`, at least the bytes that the *_workspace function of the
 * same arguments gives; 256-byte aligned; not shared by calls that may run at the same time), so any number of calls
 * may run at once and every call may be captured into a graph.  0 on success, -1 on error with vox_hip_last_error(); arguments are
 * checked on the host before anything is enqueued.  Values in device memory (lengths, parents, masks, tokens) cannot be checked there:
 * the comments say what an impossible one does, and none makes a kernel leave its buffers.
 * The last dimension of q, k, v, caches, logits, x, w is contiguous; the other strides are free and count elements.
 */
#ifndef VOX_HIP_OPS_H
#define VOX_HIP_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum vox_hip_dtype { VOX_F32 = 0, VOX_BF16 = 1, VOX_F16 = 2 };

#define VOX_TREE_MAX_NODES 256        /* nodes of one draft tree */
#define VOX_SCORES_MAX_TOP 64         /* alternatives of one row of logits */
#define VOX_I8_MAX_K 131072           /* |sum| <= 127 * 128 * K stays below 2^31 */

/* parents [batch, nodes] (-1 = the cache's end, otherwise an earlier node), n_nodes [batch] or NULL (all) ->
 * ancestors [batch, nodes, ceil(nodes / 64)]: bit j % 64 of word j / 64 of row i is set if j is i or an ancestor of i;
 * depth [batch, nodes].  Nodes that are not there (i >= n_nodes, a parent that is no earlier node and not -1, or behind such a
 * one) get no bits and depth -1. */
int vox_hip_tree_plan(const int32_t *parents, const int32_t *n_nodes, int batch, int nodes, uint64_t *ancestors, int32_t *depth,
                      int device, void *stream);

/* out[b, i, h] = sum_j p_j v_j / sum_j p_j, p_j = exp(scale * q[b, i, h] . k_j - max), over
 *   the cache's positions p of [max(0, cache_len - cap), cache_len) with window <= 0 or p > cache_len + depth[i] - window
 *   (position p lives in row p % cap of the ring), and
 *   the nodes j in ancestors[b, i] (any bit set, not only trees') with window <= 0 or depth[j] > depth[i] - window;
 * kv head = h / (heads / kv_heads).  scale is not 0 and at most 2e38 in size.  A row with depth -1 or with nothing to attend to gives zeros (lse = -inf); what masked keys and
 * values hold, NaN and infinities too, does not matter (one that a row does see may make the row's outputs infinite or NaN).  cache_len <= 0 is an empty cache.
 * Arithmetic: scores, softmax statistics and sums are f32.  bf16 and f16: every weight p_j is rounded to that type in front of its product with v (half
 * a step: 2^-8 or 2^-11 of the weighted mean of |v|), their sum is taken of the unrounded ones.  f32: where a kv head has many rows, products are taken
 * in bf16 parts and are up to 2^-21 of themselves too small.  The outputs' sums run before the division by the weights' sum: values of more than 1e28 may
 * overflow on the way. */
typedef struct vox_hip_tree_attn {
    const void *q, *k, *v;               /* [batch, nodes, heads | kv_heads, head_dim] */
    const void *k_cache, *v_cache;       /* [batch, cap, kv_heads, head_dim] */
    const int32_t *cache_len;            /* [batch] */
    const uint64_t *ancestors;           /* [batch, nodes, ceil(nodes / 64)], contiguous */
    const int32_t *depth;                /* [batch, nodes], contiguous */
    void *out;                           /* [batch, nodes, heads, head_dim]; must not overlap an input */
    float *lse;                          /* [batch, nodes, heads] contiguous: log of the sum, max added; or NULL */
    int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, kc_sb, kc_ss, kc_sh, vc_sb, vc_ss, vc_sh, o_sb, o_st, o_sh;
    int32_t dtype, batch, nodes, heads, kv_heads, head_dim, cap, window;
    float scale;
    int32_t reserved;                    /* 0 */
} vox_hip_tree_attn_t;
int64_t vox_hip_tree_attention_workspace(const vox_hip_tree_attn_t *a);      /* bytes, or -1 (reads sizes, strides and pointer alignment) */
int vox_hip_tree_attention(const vox_hip_tree_attn_t *a, void *ws, size_t ws_bytes, int device, void *stream);

/* tokens [batch, nodes]: the drafted ones; choices [batch, nodes]: the model's token behind each node; root_choice [batch]: its token
 * behind the cache.  A node is accepted if its token is what the model chose behind its parent, its ancestors are accepted, and no
 * earlier sibling has the same token.  path [batch, nodes]: the accepted nodes in order, -1 behind them; n_accepted [batch];
 * next_token [batch]: the model's choice behind the path; new_len [batch] = max(cache_len, 0) + n_accepted. */
int vox_hip_tree_accept(const int32_t *tokens, const int32_t *choices, const int32_t *root_choice, const int32_t *parents,
                        const uint64_t *ancestors, const int32_t *depth, const int32_t *cache_len, int batch, int nodes,
                        int32_t *path, int32_t *n_accepted, int32_t *next_token, int32_t *new_len, int device, void *stream);

/* Row path[b, j] of k / v [layers, batch, nodes, kv_heads, head_dim] to row (cache_len[b] + j) % cap of the caches
 * [layers, batch, cap, kv_heads, head_dim], j < n_accepted[b]; cache_len is the length BEFORE the path.  All other rows stay as they are.
 * Strides (host arrays of 4: layer, batch, row, head).  nodes <= cap.  A path entry that is no node is skipped.  The caches must not
 * overlap k and v. */
int vox_hip_tree_commit(int dtype, int layers, int batch, int nodes, int kv_heads, int head_dim, int cap, const void *k, const int64_t *k_strides,
                        const void *v, const int64_t *v_strides, void *k_cache, const int64_t *kc_strides, void *v_cache, const int64_t *vc_strides,
                        const int32_t *path, const int32_t *n_accepted, const int32_t *cache_len, int device, void *stream);

/* logits [rows, vocab] (row stride in elements) ->
 * logprob [rows, given] of tokens [rows, given] (contiguous; an id outside the vocabulary gives -inf), entropy [rows] in nats, lse [rows],
 * the `top` largest logits' indexes and log probabilities [rows, top], equal logits by the lowest index.  given = 0 / top = 0: those
 * pointers may be NULL.  A logit of -inf is a token of probability 0 (a row of nothing else: lse -inf, entropy 0, every logprob -inf);
 * a NaN makes its row's lse, entropy and logprobs NaN and counts as the largest; +inf without a NaN makes lse +inf and
 * the entropy and log probabilities NaN.  Finite logits of any size are ordinary ones (tokens switched off with the type's lowest number as well).  Sums
 * are f32. */
int64_t vox_hip_token_scores_workspace(int dtype, int64_t rows, int vocab, int top);
int vox_hip_token_scores(int dtype, const void *logits, int64_t row_stride, int64_t rows, int vocab, const int32_t *tokens, int given, int top,
                         float *logprob, float *entropy, float *lse, int32_t *top_index, float *top_logprob, void *ws, size_t ws_bytes,
                         int device, void *stream);

/* Row-wise symmetric quantisation: scale[m] = max(max_k |x[m, k]| / 127, 2^-126) in f32, q = x / scale rounded to the nearest whole
 * number, ties to even (of the exact quotient).  A row that holds an infinity or NaN gets scale NaN and zeros.  q [rows, K] contiguous. */
int vox_hip_quantize_rows_i8(int dtype, const void *x, int64_t row_stride, int64_t rows, int K, int8_t *q, float *scale, int device, void *stream);

/* y[m, n] = x_scale[m] * w_scale[n] * sum_k xq[m, k] * w[n, k] (+ bias[n]): x [rows, K] is quantised as above within the call, the sum is
 * exact, its conversion to f32 (where it is above 2^24), the two scalings, the bias and the output's type round once each.
 * w [N, K] int8 (row stride in bytes), w_scale [N] f32, bias [N] in x's type or NULL, y [rows, N] in x's type, row stride in elements. */
int64_t vox_hip_linear_i8_workspace(int dtype, int64_t rows, int K, int N, const int8_t *w, int64_t w_stride);      /* (reads w's alignment) */
int vox_hip_linear_i8(int dtype, const void *x, int64_t x_stride, int64_t rows, int K, int N, const int8_t *w, int64_t w_stride,
                      const float *w_scale, const void *bias, void *y, int64_t y_stride, void *ws, size_t ws_bytes, int device, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* VOX_HIP_OPS_H */
