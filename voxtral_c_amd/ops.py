"""Operators of a draft-verification step on torch tensors (include/vox_hip_ops.h has the definitions).

A verification pass takes several drafted tokens through the decoder at once::

    ancestors, depth = ops.tree_plan(parents, n_nodes)              # once per pass
    for every layer:
        qkv = ops.linear_i8(x, w, w_scale)                          # the nodes' rows through a matrix of 8-bit integers
        o = ops.tree_attention(q, k, v, k_cache, v_cache, cache_len, ancestors, depth)
    choices = ops.token_scores(logits, top=1).top_index
    path, n, next_token, new_len = ops.tree_accept(tokens, choices, root_choice, parents, ancestors, depth, cache_len)
    ops.tree_commit(k_all, v_all, k_caches, v_caches, path, n, cache_len)

Every function enqueues HIP kernels on torch's current stream of the tensors' device and returns without waiting; results and scratch
memory come from torch's allocator, so the calls may be captured into a graph.  Types: float32, bfloat16, float16 (one for all of a
call's tensors), int32 for lengths, tokens and tree tables, int64 for the 64-bit words of ancestor sets.  Wrong arguments raise
ValueError, what only the library finds wrong (a scale of 0, a batch beyond its grids) and a failed launch VoxError.  Sums and softmax statistics are
float32; in the 16-bit types the attention's weights are rounded to the type in front of their product with the values.  There are no
derivatives: tensors that need gradients, or carry a forward-mode tangent, are refused.
"""
import ctypes as C
import operator
import struct
import warnings
from collections import namedtuple

import torch
from torch.autograd.forward_ad import unpack_dual

from . import VoxError, hip

try:
    from . import _ops_call as _call
except ImportError as e:                                               # not built, or built for another interpreter or torch
    warnings.warn(f"{e}: the operators' calls go over ctypes (the same kernels, more host time per call)", RuntimeWarning, stacklevel=2)

    class _call:
        """Takes nothing: every call is made here."""

        tree_plan = tree_attention = tree_accept = tree_commit = token_scores = quantize_rows_i8 = linear_i8 = bind = staticmethod(lambda *args: None)

MAX_NODES = 256
MAX_TOP = 64
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_I32 = torch.int32

_p, _i, _q = C.c_void_p, C.c_int, C.c_int64
_ATTN = struct.Struct("10P18q8ifi")
hip.vox_hip_tree_plan.argtypes = [_p, _p, _i, _i, _p, _p, _i, _p]
hip.vox_hip_tree_attention_workspace.argtypes = [C.c_char_p]
hip.vox_hip_tree_attention_workspace.restype = _q
hip.vox_hip_tree_attention.argtypes = [C.c_char_p, _p, C.c_size_t, _i, _p]
hip.vox_hip_tree_accept.argtypes = [_p] * 7 + [_i, _i] + [_p] * 4 + [_i, _p]
hip.vox_hip_tree_commit.argtypes = [_i] * 7 + [_p, C.POINTER(_q)] * 4 + [_p] * 3 + [_i, _p]
hip.vox_hip_token_scores_workspace.argtypes = [_i, _q, _i, _i]
hip.vox_hip_token_scores_workspace.restype = _q
hip.vox_hip_token_scores.argtypes = [_i, _p, _q, _q, _i, _p, _i, _i] + [_p] * 6 + [C.c_size_t, _i, _p]
hip.vox_hip_quantize_rows_i8.argtypes = [_i, _p, _q, _q, _i, _p, _p, _i, _p]
hip.vox_hip_linear_i8_workspace.argtypes = [_i, _q, _i, _i, _p, _q]
hip.vox_hip_linear_i8_workspace.restype = _q
hip.vox_hip_linear_i8.argtypes = [_i, _p, _q, _q, _i, _i, _p, _q, _p, _p, _p, _q, _p, C.c_size_t, _i, _p]
_Strides = _q * 4


def _error(who):
    raise VoxError(f"{who}: {hip.vox_hip_last_error().decode()}")


def _derivatives(who, name, t):
    """Refuses what a backward pass, or forward mode, would want a derivative of."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{who}: {name} needs gradients: there is no backward pass (use torch.no_grad())")
    if torch._C._is_fwd_grad_enabled() and unpack_dual(t).tangent is not None:
        raise ValueError(f"{who}: {name} has a tangent: there is no forward-mode derivative (use unpack_dual(..).primal)")


def _float_args(who, *named):
    """`named`: name, tensor, shape, name, .. .  One floating type of _DTYPES, the given shapes, a contiguous last dimension; returns the type's number."""
    dtype = named[1].dtype
    for i in range(0, len(named), 3):
        t, shape = named[i + 1], named[i + 2]
        if t.dtype is not dtype or t.shape != shape or (t.stride(-1) != 1 and shape[-1] > 1) or dtype not in _DTYPES:
            name = named[i]
            if dtype not in _DTYPES:
                raise ValueError(f"{who}: {name} is {dtype}: float32, bfloat16 or float16 are supported")
            if t.dtype != dtype:
                raise ValueError(f"{who}: {name} is {t.dtype}, {named[0]} is {dtype}: one type is needed")
            if t.shape != shape:
                raise ValueError(f"{who}: {name} has the shape {tuple(t.shape)}: {tuple(shape)} is needed")
            raise ValueError(f"{who}: the last dimension of {name} is not contiguous")
        _derivatives(who, named[i], t)
    return _DTYPES[dtype]


def _table(who, name, t, shape, dtype=_I32):
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{who}: {name} is {t.dtype} {tuple(t.shape)}: {dtype} {tuple(shape)} is needed")
    return t if t.is_contiguous() else t.contiguous()


def _sizes(who, *tensors):
    """The library counts sizes in 32 bits, and ctypes would hand it the low ones of a larger number without a word."""
    for t in tensors:
        if max(t.shape, default=0) > 0x7fffffff:
            raise ValueError(f"{who}: shape {tuple(t.shape)}: sizes of 2^31 and more are not supported")


def _whole(who, name, number):
    """A whole number of any kind (Python's, numpy's, a tensor of one) as Python's own."""
    try:
        return operator.index(number)
    except TypeError:
        raise ValueError(f"{who}: {name} {number!r}: a whole number is needed") from None


def _device(who, *tensors):
    """The tensors' one GPU, as its number; all of a call's tensors are seen here, and what lies in their memory has to be their values."""
    d = tensors[0].get_device()
    for t in tensors:
        if t.is_neg():
            raise ValueError(f"{who}: a tensor of the shape {tuple(t.shape)} is negated lazily (use resolve_neg())")
    for t in tensors:
        if t.get_device() != d or d < 0:
            raise ValueError(f"{who}: tensors on {tensors[0].device} and {t.device}: " + ("one device is needed" if t.device != tensors[0].device else
                                                                                            "a GPU is needed (there is no CPU path)"))
    return d


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)      # (what current_stream gives, without the object around it)


def _stream(device):
    return _raw_stream(device) if _raw_stream else torch.cuda.current_stream(device).cuda_stream


# The compiled calls (csrc/vox_ops_call.cpp) take what is in order; what they hand back as None is done or refused here.
_call.bind(_raw_stream or _stream, *(C.cast(getattr(hip, "vox_hip_" + n), _p).value for n in (
    "tree_plan", "tree_attention_workspace", "tree_attention", "tree_accept", "tree_commit", "token_scores_workspace", "token_scores",
    "quantize_rows_i8", "linear_i8_workspace", "linear_i8")))


def _nodes(who, shape):
    if len(shape) < 2 or shape[1] > MAX_NODES:
        raise ValueError(f"{who}: shape {tuple(shape)}: [batch, nodes, ..] with at most {MAX_NODES} nodes is needed")


def tree_plan(parents, n_nodes=None):
    """Ancestor sets int64 [batch, nodes, ceil(nodes / 64)] and depths int32 [batch, nodes] of draft trees: parents int32 [batch, nodes], -1 for
    the cache's end, otherwise an earlier node; n_nodes int32 [batch] where trees are shorter than the padded width."""
    done = _call.tree_plan(parents, n_nodes)
    if done is not None:
        return done
    who = "tree_plan"
    _sizes(who, parents)
    _nodes(who, parents.shape)
    B, T = parents.shape if parents.dim() == 2 else (-1, -1)
    parents = _table(who, "parents", parents, (B, T))
    if n_nodes is not None:
        n_nodes = _table(who, "n_nodes", n_nodes, (B,))
    d = _device(who, parents, *(() if n_nodes is None else (n_nodes,)))
    ancestors = parents.new_empty((B, T, (T + 63) // 64), dtype=torch.int64)
    depth = torch.empty_like(parents)
    if hip.vox_hip_tree_plan(parents.data_ptr(), None if n_nodes is None else n_nodes.data_ptr(), B, T, ancestors.data_ptr(), depth.data_ptr(), d, _stream(d)):
        _error(who)
    return ancestors, depth


def tree_attention(q, k, v, k_cache, v_cache, cache_len, ancestors, depth, scale=None, window=0, return_lse=False):
    """Attention of draft nodes over a ring cache and their own ancestors: q [batch, nodes, heads, dim], k and v [batch, nodes, kv_heads, dim],
    caches [batch, cap, kv_heads, dim] (position p in row p % cap), cache_len int32 [batch], the tables of tree_plan (or any other mask of
    that form).  window <= 0: none, otherwise a node sees positions above its own - window.  Rows that see nothing are zeros.
    Returns out like q, with return_lse (out, float32 [batch, nodes, heads])."""
    done = _call.tree_attention(q, k, v, k_cache, v_cache, cache_len, ancestors, depth, scale, window, return_lse)
    if done is not None:
        return done
    who = "tree_attention"
    _sizes(who, q, k, k_cache)
    if q.dim() != 4 or k_cache.dim() != 4 or k.dim() != 4:
        raise ValueError(f"{who}: q, k and the caches have 4 dimensions: got {q.dim()}, {k.dim()}, {k_cache.dim()}")
    B, T, H, D = q.shape
    cap, Hk = k_cache.shape[1], k.shape[2]
    _nodes(who, q.shape)
    if Hk < 1 or H % Hk or not 1 <= D <= 256 or cap < 1:
        raise ValueError(f"{who}: {H} heads over {Hk} kv heads of {D} (at most 256), a cache of {cap} rows")
    window = _whole(who, "window", window)
    try:
        scale = D ** -0.5 if scale is None else float(scale * 1.0)
    except TypeError:
        raise ValueError(f"{who}: scale {scale!r}: a number is needed") from None
    cache = (B, cap, Hk, D)
    number = _float_args(who, "q", q, q.shape, "k", k, (B, T, Hk, D), "v", v, (B, T, Hk, D), "k_cache", k_cache, cache, "v_cache", v_cache, cache)
    cache_len = _table(who, "cache_len", cache_len, (B,))
    ancestors = _table(who, "ancestors", ancestors, (B, T, (T + 63) // 64), torch.int64)
    depth = _table(who, "depth", depth, (B, T))
    d = _device(who, q, k, v, k_cache, v_cache, cache_len, ancestors, depth)
    out = q.new_empty((B, T, H, D))
    lse = q.new_empty((B, T, H), dtype=torch.float32) if return_lse else None
    args = _ATTN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), cache_len.data_ptr(), ancestors.data_ptr(), depth.data_ptr(),
                      out.data_ptr(), 0 if lse is None else lse.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *k_cache.stride()[:3], *v_cache.stride()[:3],
                      T * H * D, H * D, D, number, B, T, H, Hk, D, cap, max(-1, min(window, 0x7fffffff)), scale, 0)
    need = hip.vox_hip_tree_attention_workspace(args)
    ws = q.new_empty(need, dtype=torch.uint8) if need > 0 else None
    if need < 0 or hip.vox_hip_tree_attention(args, None if ws is None else ws.data_ptr(), need, d, _stream(d)):
        _error(who)
    return (out, lse) if return_lse else out


def tree_accept(tokens, choices, root_choice, parents, ancestors, depth, cache_len):
    """The drafted path that the model agrees with: tokens and choices (the model's token behind each node) int32 [batch, nodes], root_choice
    (its token behind the cache) int32 [batch].  Returns path int32 [batch, nodes] (-1 behind the accepted nodes), their number,
    the model's token behind the path, and the cache's new length, int32 [batch] each."""
    done = _call.tree_accept(tokens, choices, root_choice, parents, ancestors, depth, cache_len)
    if done is not None:
        return done
    who = "tree_accept"
    _sizes(who, tokens)
    _nodes(who, tokens.shape)
    B, T = tokens.shape if tokens.dim() == 2 else (-1, -1)
    if T == 0:
        raise ValueError(f"{who}: no nodes")
    tokens, choices = _table(who, "tokens", tokens, (B, T)), _table(who, "choices", choices, (B, T))
    parents, depth = _table(who, "parents", parents, (B, T)), _table(who, "depth", depth, (B, T))
    root_choice, cache_len = _table(who, "root_choice", root_choice, (B,)), _table(who, "cache_len", cache_len, (B,))
    ancestors = _table(who, "ancestors", ancestors, (B, T, (T + 63) // 64), torch.int64)
    d = _device(who, tokens, choices, root_choice, parents, ancestors, depth, cache_len)
    path = torch.empty_like(tokens)
    n, after, new_len = root_choice.new_empty((3, B)).unbind()
    if hip.vox_hip_tree_accept(tokens.data_ptr(), choices.data_ptr(), root_choice.data_ptr(), parents.data_ptr(), ancestors.data_ptr(), depth.data_ptr(),
                               cache_len.data_ptr(), B, T, path.data_ptr(), n.data_ptr(), after.data_ptr(), new_len.data_ptr(), d, _stream(d)):
        _error(who)
    return path, n, after, new_len


def tree_commit(k, v, k_cache, v_cache, path, n_accepted, cache_len):
    """Files the path's keys and values into the ring caches, in place: k and v [layers, batch, nodes, kv_heads, dim], caches [layers, batch, cap,
    kv_heads, dim] (or all four without the layers), cache_len the length before the path.  The caches' versions rise, as by torch's own in-place operations."""
    who = "tree_commit"
    if k.dim() == 4:
        k, v, k_cache, v_cache = k[None], v[None], k_cache[None], v_cache[None]
    if _call.tree_commit(k, v, k_cache, v_cache, path, n_accepted, cache_len):
        return
    _sizes(who, k, k_cache)
    if k.dim() != 5 or k_cache.dim() != 5:
        raise ValueError(f"{who}: k {tuple(k.shape)}, k_cache {tuple(k_cache.shape)}: [layers,] batch, rows, kv_heads, dim are needed")
    L, B, T, Hk, D = k.shape
    cap = k_cache.shape[2]
    _nodes(who, k.shape[1:])
    if cap < T:
        raise ValueError(f"{who}: a ring of {cap} rows does not hold a path of {T} nodes")
    number = _float_args(who, "k", k, k.shape, "v", v, k.shape, "k_cache", k_cache, (L, B, cap, Hk, D), "v_cache", v_cache, (L, B, cap, Hk, D))
    path, n_accepted, cache_len = _table(who, "path", path, (B, T)), _table(who, "n_accepted", n_accepted, (B,)), _table(who, "cache_len", cache_len, (B,))
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
            raise ValueError(f"{who}: {name} is an expanded tensor: its rows share memory")
    d = _device(who, k, v, k_cache, v_cache, path, n_accepted, cache_len)
    if hip.vox_hip_tree_commit(number, L, B, T, Hk, D, cap, k.data_ptr(), _Strides(*k.stride()[:4]), v.data_ptr(), _Strides(*v.stride()[:4]),
                               k_cache.data_ptr(), _Strides(*k_cache.stride()[:4]), v_cache.data_ptr(), _Strides(*v_cache.stride()[:4]),
                               path.data_ptr(), n_accepted.data_ptr(), cache_len.data_ptr(), d, _stream(d)):
        _error(who)
    for t in (k_cache, v_cache):                                       # what autograd has saved of them is theirs no longer
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


TokenScores = namedtuple("TokenScores", "logprob entropy lse top_index top_logprob")


def token_scores(logits, tokens=None, top=0):
    """Scores of rows of logits [rows, vocab]: log probabilities of `tokens` int32 [rows, given] (or [rows]), the distribution's entropy and
    log-sum [rows], and the `top` largest logits' indexes and log probabilities [rows, top], equal ones by the lowest index.  An id outside
    the vocabulary scores -inf."""
    done = _call.token_scores(logits, tokens, top)
    if done is not None:
        return TokenScores(*done)
    who = "token_scores"
    _sizes(who, logits, *(() if tokens is None else (tokens,)))
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"{who}: logits have the shape {tuple(logits.shape)}: [rows, vocab] is needed")
    R, V = logits.shape
    number, top = _float_args(who, "logits", logits, logits.shape), _whole(who, "top", top)
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"{who}: top {top} of {V} (at most {MAX_TOP})")
    shape = (R, 0)
    if tokens is not None:
        shape = (R, tokens.shape[1]) if tokens.dim() == 2 else (R,)
        tokens = _table(who, "tokens", tokens, shape)
    d = _device(who, logits) if tokens is None else _device(who, logits, tokens)
    new, f32 = logits.new_empty, torch.float32
    logprob, entropy, lse, top_index, top_logprob = new(shape, dtype=f32), new((R,), dtype=f32), new((R,), dtype=f32), new((R, top), dtype=_I32), new((R, top), dtype=f32)
    need = hip.vox_hip_token_scores_workspace(number, R, V, top)
    ws = new(need, dtype=torch.uint8) if need > 0 else None
    given = 0 if tokens is None else 1 if len(shape) == 1 else shape[1]
    if need < 0 or hip.vox_hip_token_scores(number, logits.data_ptr(), logits.stride(0), R, V, None if tokens is None else tokens.data_ptr(), given, top,
                                            logprob.data_ptr(), entropy.data_ptr(), lse.data_ptr(), top_index.data_ptr(), top_logprob.data_ptr(),
                                            None if ws is None else ws.data_ptr(), need, d, _stream(d)):
        _error(who)
    return TokenScores(logprob, entropy, lse, top_index, top_logprob)


def quantize_rows_i8(x):
    """x [rows, K] -> (int8 [rows, K], float32 scales [rows]): scale = largest magnitude / 127, whole numbers to nearest, ties to even.  With a
    weight matrix [outputs, inputs] this gives linear_i8's w and w_scale."""
    done = _call.quantize_rows_i8(x)
    if done is not None:
        return done
    who = "quantize_rows_i8"
    _sizes(who, x)
    if x.dim() != 2 or not 1 <= x.shape[1] <= 131072:
        raise ValueError(f"{who}: x has the shape {tuple(x.shape)}: [rows, K] with K of 1 to 131072 is needed")
    number = _float_args(who, "x", x, x.shape)
    d = _device(who, x)
    q, scale = x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[0], dtype=torch.float32)
    if hip.vox_hip_quantize_rows_i8(number, x.data_ptr(), x.stride(0), x.shape[0], x.shape[1], q.data_ptr(), scale.data_ptr(), d, _stream(d)):
        _error(who)
    return q, scale


def linear_i8(x, w, w_scale, bias=None):
    """y [rows, outputs] in x's type = x [rows, inputs], quantised row by row as quantize_rows_i8 does, times w int8 [outputs, inputs] with one float32
    scale per output, plus bias [outputs] in x's type.  The sum of the whole numbers is exact."""
    done = _call.linear_i8(x, w, w_scale, bias)
    if done is not None:
        return done
    who = "linear_i8"
    _sizes(who, x, w)
    if x.dim() != 2 or not 1 <= x.shape[1] <= 131072 or w.dim() != 2:
        raise ValueError(f"{who}: x has the shape {tuple(x.shape)}, w {tuple(w.shape)}: [rows, K] and [outputs, K] with K of 1 to 131072 are needed")
    M, K = x.shape
    N = w.shape[0]
    number = _float_args(who, "x", x, x.shape) if bias is None else _float_args(who, "x", x, x.shape, "bias", bias, (N,))
    if w.dtype != torch.int8 or w.shape[1] != K or (w.stride(1) != 1 and K > 1):
        raise ValueError(f"{who}: w is {w.dtype} {tuple(w.shape)}: int8 {(N, K)} with contiguous rows is needed")
    w_scale = _table(who, "w_scale", w_scale, (N,), torch.float32)
    _derivatives(who, "w_scale", w_scale)
    d = _device(who, x, w, w_scale, *(() if bias is None else (bias,)))
    y = x.new_empty((M, N))
    wp, wst = w.data_ptr(), w.stride(0)
    need = hip.vox_hip_linear_i8_workspace(number, M, K, N, wp, wst)
    ws = x.new_empty(need, dtype=torch.uint8) if need > 0 else None
    if need < 0 or hip.vox_hip_linear_i8(number, x.data_ptr(), x.stride(0), M, K, N, wp, wst, w_scale.data_ptr(),
                                         None if bias is None else bias.data_ptr(), y.data_ptr(), N, None if ws is None else ws.data_ptr(), need, d, _stream(d)):
        _error(who)
    return y
