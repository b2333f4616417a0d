"""CPU: what the draft-verification operators refuse at the edges of their arguments, and how they are built and loaded."""
import os
import shutil
import subprocess
import sys

import pytest
import torch

from conftest import ROOT
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


def make_plan(*settings, path=None):
    """What `make all` would run from nothing."""
    r = subprocess.run(["make", "-n", "-B", "all", *settings], cwd=os.path.join(ROOT, "voxtral_c_amd"), capture_output=True, text=True, env={**os.environ, **({"PATH": path} if path else {})})
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_the_libraries_build_without_python_or_torch(tmp_path):
    """The compiled calls need this interpreter's headers and its torch; the libraries need hipcc and a C compiler, and `make all` ends with them where that is all there is."""
    full = make_plan()
    assert "-o libvoxhip.so" in full and "-o libvoxtral.so" in full and "-o _ops_call.so" in full
    for tool in ("make", "sh"):
        os.symlink(shutil.which(tool), tmp_path / tool)
    for plan in (make_plan("TORCH="), make_plan("PYINC=/nowhere"), make_plan(path=str(tmp_path))):        # no torch, no headers, no python3 at all
        assert "-o libvoxhip.so" in plan and "-o libvoxtral.so" in plan and "-o _ops_call.so" not in plan


def test_the_operators_load_without_their_compiled_calls():
    """Without the module (not built, or built for another torch) the same calls go over ctypes, checks and all, and a warning says so."""
    code = """
import sys, warnings
sys.modules["voxtral_c_amd._ops_call"] = None                          # the import fails
import torch
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter("always")
    from voxtral_c_amd import ops
assert any("_ops_call" in str(w.message) for w in seen)
t = torch.zeros(1, 3, dtype=torch.int32)
for call in (lambda: ops.tree_plan(t), lambda: ops.quantize_rows_i8(torch.zeros(2, 3)), lambda: ops.token_scores(torch.zeros(2, 3)),
             lambda: ops.linear_i8(torch.zeros(2, 3), torch.zeros(4, 3, dtype=torch.int8), torch.zeros(4))):
    try:
        call()
    except ValueError as e:
        assert "a GPU is needed" in str(e)
    else:
        raise AssertionError
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.stdout.strip() == "fine", r.stderr


@pytest.mark.parametrize("scale,fine", [(1.0, True), (-1e38, True), (1e38, True), (3e38, False), (-2.5e38, False), (0.0, False), (float("inf"), False), (float("nan"), False), (1e-30, True)])
def test_tree_attention_takes_scales_whose_base_2_form_is_finite(scale, fine):
    """The softmax runs in base 2: scale * log2(e) has to be a number, or a score of 0 would become NaN."""
    args = ops._ATTN.pack(*[4096] * 10, *[8] * 18, 0, 1, 2, 4, 2, 64, 8, 0, scale, 0)
    assert (ops.hip.vox_hip_tree_attention_workspace(args) >= 0) == fine
    assert fine or "scale" in ops.hip.vox_hip_last_error().decode()


def test_sizes_of_nothing_are_refused_by_name():
    z, n, t, a = torch.zeros, torch.zeros(1, dtype=I32), torch.zeros(1, 2, dtype=I32), torch.zeros(1, 2, 1, dtype=torch.int64)
    with pytest.raises(ValueError, match="tree_attention: 2 heads over 1 kv heads of 0"):
        ops.tree_attention(z(1, 2, 2, 0), z(1, 2, 1, 0), z(1, 2, 1, 0), z(1, 5, 1, 0), z(1, 5, 1, 0), n, a, t)
    with pytest.raises(ValueError, match="window 9.5: a whole number"):
        ops.tree_attention(z(1, 2, 2, 4), z(1, 2, 1, 4), z(1, 2, 1, 4), z(1, 5, 1, 4), z(1, 5, 1, 4), n, a, t, window=9.5)
    with pytest.raises(ValueError, match="top 1.5: a whole number"):
        ops.token_scores(z(2, 3), None, 1.5)
