"""CPU: what the draft-verification operators refuse at the edges of their arguments, and how they are built and loaded."""
import pytest
import torch

from voxtral_c_amd import ops

I32 = torch.int32


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")              # (shapes and types without memory)


FAR = 2 ** 32 + 3                                                      # a size whose low 32 bits are an ordinary one


def attention_of(B, T, H, D, Hk, cap):
    m = meta
    return (m(B, T, H, D), m(B, T, Hk, D), m(B, T, Hk, D), m(B, cap, Hk, D), m(B, cap, Hk, D), m(B, dtype=I32), m(B, T, (T + 63) // 64, dtype=torch.int64), m(B, T, dtype=I32))


def commit_of(L, B, T, Hk, D, cap):
    k, c = meta(L, B, T, Hk, D), meta(L, B, cap, Hk, D)
    return k, k, c, c, meta(B, T, dtype=I32), meta(B, dtype=I32), meta(B, dtype=I32)


def accept_of(B, T):
    t, r = meta(B, T, dtype=I32), meta(B, dtype=I32)
    return t, t, r, t, meta(B, T, 1, dtype=torch.int64), t, r


@pytest.mark.parametrize("call,args", [
    ("tree_plan", (meta(FAR, 1, dtype=I32),)), ("tree_plan", (meta(FAR, 0, dtype=I32),)), ("tree_accept", accept_of(FAR, 1)),
    ("tree_attention", attention_of(FAR, 1, 1, 1, 1, 4)), ("tree_attention", attention_of(1, 1, FAR, 1, 1, 4)), ("tree_attention", attention_of(1, 1, 1, 1, 1, FAR)),
    ("tree_commit", commit_of(FAR, 1, 1, 1, 1, 4)), ("tree_commit", commit_of(1, FAR, 1, 1, 1, 4)), ("tree_commit", commit_of(1, 1, 1, FAR, 1, 4)),
    ("tree_commit", commit_of(1, 1, 1, 1, FAR, 4)), ("tree_commit", commit_of(1, 1, 1, 1, 1, FAR)),
    ("token_scores", (meta(1, FAR),)), ("token_scores", (meta(FAR, 5),)), ("token_scores", (meta(1, 5), meta(1, FAR, dtype=I32))),
    ("quantize_rows_i8", (meta(FAR, 2),)), ("linear_i8", (meta(1, 2), meta(FAR, 2, dtype=torch.int8), meta(FAR))), ("linear_i8", (meta(FAR, 2), meta(1, 2, dtype=torch.int8), meta(1))),
], ids=lambda a: a if isinstance(a, str) else "x".join("-".join(map(str, t.shape)) for t in a[:1]))
def test_sizes_beyond_31_bits_are_refused(call, args):
    """The library counts sizes in 32 bits: a larger one is refused, never cut to its low bits."""
    with pytest.raises(ValueError, match=f"{call}: .*2\\^31"):
        getattr(ops, call)(*args)


def tangent(t):
    return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))


def test_forward_mode_tangents_are_refused():
    """There are no derivatives in either direction: a dual tensor's tangent would be lost without a word."""
    z = torch.zeros
    x, w, s, q, k, c = z(2, 8), z(3, 8, dtype=torch.int8), z(3), z(1, 2, 2, 4), z(1, 2, 1, 4), z(1, 5, 1, 4)
    n, t, a = z(1, dtype=I32), z(1, 2, dtype=I32), z(1, 2, 1, dtype=torch.int64)
    calls = [(ops.quantize_rows_i8, [x], [0]), (ops.linear_i8, [x, w, s, s], [0, 2, 3]), (ops.token_scores, [x], [0]), (ops.tree_attention, [q, k, k, c, c, n, a, t], [0, 1, 2, 3, 4]),
             (ops.tree_commit, [k[None], k[None], c[None], c[None], t, n, n], [0, 1, 2, 3]), (ops.tree_commit, [k, k, c, c, t, n, n], [0, 1, 2, 3])]
    for f, args, places in calls:
        for i in places:
            with torch.autograd.forward_ad.dual_level():
                dual = [*args[:i], tangent(args[i]), *args[i + 1:]]
                for mode in (torch.enable_grad, torch.no_grad):        # (no_grad does not switch forward mode off)
                    with mode(), pytest.raises(ValueError, match="tangent"):
                        f(*dual)
                with torch.inference_mode(), pytest.raises(ValueError, match="a GPU is needed"):
                    f(*dual)
            with pytest.raises(ValueError, match="a GPU is needed"):
                f(*args)


def test_lazily_negated_tensors_are_refused():
    """Such a tensor's memory holds the values with the other sign: it is not read (or, a cache, written) as it is."""
    z = torch.zeros
    x, w, s, q, k, c = z(2, 8), z(3, 8, dtype=torch.int8), z(3), z(1, 2, 2, 4), z(1, 2, 1, 4), z(1, 5, 1, 4)
    n, t, a = z(1, dtype=I32), z(1, 2, dtype=I32), z(1, 2, 1, dtype=torch.int64)
    calls = [(ops.quantize_rows_i8, [x]), (ops.linear_i8, [x, w, s, s]), (ops.token_scores, [x, z(2, 1, dtype=I32)]), (ops.tree_attention, [q, k, k, c, c, n, a, t]),
             (ops.tree_commit, [k[None], k[None], c[None], c[None], t, n, n]), (ops.tree_commit, [k, k, c, c, t, n, n]), (ops.tree_plan, [t, n]), (ops.tree_accept, [t, t, n, t, a, t, n])]
    for f, args in calls:
        for i in range(len(args)):
            with pytest.raises(ValueError, match="negated"):
                f(*args[:i], torch._neg_view(args[i]), *args[i + 1:])
            with pytest.raises(ValueError, match="a GPU is needed"):
                f(*args[:i], torch._neg_view(args[i]).resolve_neg(), *args[i + 1:])
