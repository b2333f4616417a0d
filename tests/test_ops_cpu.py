"""CPU: the draft-verification operators' surface - exported symbols, and what they refuse before anything reaches a GPU."""
import ctypes as C
import os
import re

import pytest
import torch

from conftest import ROOT
from test_host_cpu import exported

import voxtral_c_amd as v
from voxtral_c_amd import ops

I32 = torch.int32


def test_every_operator_is_exported():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "vox_hip_ops.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(vox_hip_[a-z0-9_]+)\s*\(", text))
    assert len(declared) == 10 and not declared - exported("libvoxhip.so")


def zeros(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def attn_args(B=2, T=3, H=4, Hk=2, D=64, cap=16, dtype=torch.float32):
    return dict(q=zeros(B, T, H, D, dtype=dtype), k=zeros(B, T, Hk, D, dtype=dtype), v=zeros(B, T, Hk, D, dtype=dtype), k_cache=zeros(B, cap, Hk, D, dtype=dtype),
                v_cache=zeros(B, cap, Hk, D, dtype=dtype), cache_len=zeros(B, dtype=I32), ancestors=zeros(B, T, 1, dtype=torch.int64), depth=zeros(B, T, dtype=I32))


@pytest.mark.parametrize("change,message", [
    (dict(q=zeros(2, 3, 4, 64, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(q=zeros(2, 3, 4, 64, dtype=torch.bfloat16)), "one type"),
    (dict(q=zeros(2, 3, 5, 64)), "5 heads over 2"),
    (dict(q=zeros(2, 3, 256)), "4 dimensions"),
    (dict(k=zeros(2, 4, 2, 64)), "shape"),
    (dict(v_cache=zeros(2, 15, 2, 64)), "shape"),
    (dict(k=zeros(2, 3, 64, 2).transpose(2, 3)), "not contiguous"),
    (dict(q=zeros(2, 3, 4, 64).requires_grad_()), "no backward"),
    (dict(cache_len=zeros(2, dtype=torch.int64)), "cache_len"),
    (dict(ancestors=zeros(2, 3, 2, dtype=torch.int64)), "ancestors"),
    (dict(depth=zeros(2, 4, dtype=I32)), "depth"),
    (dict(), "a GPU is needed"),
])
def test_tree_attention_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        ops.tree_attention(**{**attn_args(), **change})


def test_tree_attention_refuses_large_trees_and_heads():
    with pytest.raises(ValueError, match="256 nodes"):
        ops.tree_attention(**attn_args(T=257))
    with pytest.raises(ValueError, match="at most 256"):
        ops.tree_attention(**attn_args(D=257))


def test_tree_tables_refuse():
    with pytest.raises(ValueError, match="256 nodes"):
        ops.tree_plan(zeros(1, 257, dtype=I32))
    with pytest.raises(ValueError, match="parents"):
        ops.tree_plan(zeros(1, 3))
    with pytest.raises(ValueError, match="n_nodes"):
        ops.tree_plan(zeros(2, 3, dtype=I32), zeros(3, dtype=I32))
    with pytest.raises(ValueError, match="parents"):
        ops.tree_plan(zeros(2, 3, 1, dtype=I32))
    t, r, m = zeros(2, 3, dtype=I32), zeros(2, dtype=I32), zeros(2, 3, 1, dtype=torch.int64)
    with pytest.raises(ValueError, match="root_choice"):
        ops.tree_accept(t, t, t, t, m, t, r)
    with pytest.raises(ValueError, match="choices"):
        ops.tree_accept(t, t.long(), r, t, m, t, r)
    with pytest.raises(ValueError, match="no nodes"):
        ops.tree_accept(t[:, :0], t[:, :0], r, t[:, :0], m[:, :0], t[:, :0], r)
    with pytest.raises(ValueError, match="GPU"):
        ops.tree_accept(t, t, r, t, m, t, r)


def test_tree_commit_refuses():
    k, c, path, r = zeros(5, 2, 3, 2, 8), zeros(5, 2, 16, 2, 8), zeros(2, 3, dtype=I32), zeros(2, dtype=I32)
    for args, message in (((k, k, c[:, :, :2], c[:, :, :2], path, r, r), "does not hold"), ((k, k[:4], c, c, path, r, r), "shape"), ((k, k, c, c.half(), path, r, r), "one type"),
                          ((k, k, c, c[:, :1].expand(5, 2, 16, 2, 8), path, r, r), "share memory"), ((k, k, c, c, path, path, r), "n_accepted"),
                          ((k[0, 0], k[0, 0], c, c, path, r, r), "are needed"), ((k, k, c, c, path, r, r), "GPU")):
        with pytest.raises(ValueError, match=message):
            ops.tree_commit(*args)


def test_token_scores_refuses():
    x, t = zeros(4, 100), zeros(4, 2, dtype=I32)
    for args, message in (((x[0], t), "rows, vocab"), ((x.double(), t), "float32"), ((x, t.long()), "tokens"), ((x, t[:3]), "tokens"), ((x, t, 65), "top"), ((x, t, -1), "top"),
                          ((x[:, :10].contiguous(), t, 11), "top"), ((x.t(), zeros(100, 2, dtype=I32)), "not contiguous"), ((zeros(4, 0), None), "rows, vocab"), ((x, t[0, 0]), "tokens"), ((x, t[None]), "tokens"), ((x, t, 3), "GPU")):
        with pytest.raises(ValueError, match=message):
            ops.token_scores(*args)


def test_linear_i8_refuses():
    x, w, s = zeros(4, 100), zeros(7, 100, dtype=torch.int8), zeros(7)
    for args, message in (((x[0], w, s), "rows, K"), ((x.double(), w, s), "float32"), ((x, w.float(), s), "int8"), ((x, w[:, :50], s), "int8"), ((x, w, s.half()), "w_scale"),
                          ((x, w, s[:6]), "w_scale"), ((x, w, s, zeros(6)), "bias"), ((x, w, s, zeros(7).half()), "bias"), ((x.t(), zeros(7, 4, dtype=torch.int8), s), "not contiguous"),
                          ((zeros(1, 131073), zeros(1, 131073, dtype=torch.int8), s[:1]), "131072"), ((x, w, s), "GPU")):
        with pytest.raises(ValueError, match=message):
            ops.linear_i8(*args)
    with pytest.raises(ValueError, match="gradients"):
        ops.linear_i8(x, w, s.requires_grad_())
    for x, message in ((zeros(3), "rows, K"), (zeros(3, 0), "rows, K"), (zeros(2, 3, dtype=torch.int32), "float32"), (zeros(2, 3), "GPU")):
        with pytest.raises(ValueError, match=message):
            ops.quantize_rows_i8(x)


def test_c_entries_refuse_before_any_launch():
    """Wrong sizes, null pointers and missing workspace come back as -1 with a message; none of these calls needs a GPU."""
    err = lambda: v.hip.vox_hip_last_error().decode()  # noqa: E731
    fake = 4096
    assert v.hip.vox_hip_tree_plan(fake, None, 1, 257, fake, fake, 0, None) == -1 and "256" in err()
    assert v.hip.vox_hip_tree_plan(None, None, 1, 4, fake, fake, 0, None) == -1 and "null" in err()
    assert v.hip.vox_hip_tree_plan(None, None, 0, 4, None, None, 0, None) == 0
    assert v.hip.vox_hip_tree_accept(*[fake] * 6, None, 1, 4, *[fake] * 4, 0, None) == -1 and "null" in err()
    st, bad = ops._Strides(0, 0, 8, 8), ops._Strides(0, 0, -8, 8)
    assert v.hip.vox_hip_tree_commit(0, 1, 1, 4, 1, 8, 3, fake, st, fake, st, fake, st, fake, st, fake, fake, fake, 0, None) == -1 and "does not hold" in err()
    assert v.hip.vox_hip_tree_commit(0, 1, 1, 4, 1, 8, 9, fake, st, fake, bad, fake, st, fake, st, fake, fake, fake, 0, None) == -1 and "stride" in err()
    assert v.hip.vox_hip_tree_commit(7, 1, 1, 4, 1, 8, 9, fake, st, fake, st, fake, st, fake, st, fake, fake, fake, 0, None) == -1 and "dtype" in err()
    pack = lambda **kw: ops._ATTN.pack(*[kw.get("p", fake)] * 10, *[kw.get("s", 8)] * 18, kw.get("dtype", 0), kw.get("batch", 1), kw.get("nodes", 2), kw.get("heads", 4),  # noqa: E731
                                       kw.get("kv", 2), kw.get("dim", 64), kw.get("cap", 8), 0, 1.0, kw.get("reserved", 0))
    for kw, text in ((dict(dtype=3), "dtype"), (dict(nodes=257), "nodes"), (dict(heads=5), "heads"), (dict(kv=0), "heads"), (dict(dim=0), "head_dim"), (dict(dim=257), "head_dim"),
                     (dict(cap=0), "cache"), (dict(batch=65536), "batch"), (dict(reserved=1), "reserved")):
        assert v.hip.vox_hip_tree_attention_workspace(pack(**kw)) == -1 and text in err(), kw
        assert v.hip.vox_hip_tree_attention(pack(**kw), None, 0, 0, None) == -1
    assert v.hip.vox_hip_tree_attention(pack(p=0), None, 0, 0, None) == -1 and "null" in err()
    assert v.hip.vox_hip_tree_attention(pack(s=-1), None, 0, 0, None) == -1 and "stride" in err()
    assert v.hip.vox_hip_token_scores_workspace(0, 4, 100, 65) == -1 and "top" in err()
    need = v.hip.vox_hip_token_scores_workspace(0, 1, 131072, 8)
    assert need > 0
    score = lambda ws, n: v.hip.vox_hip_token_scores(0, fake, 131072, 1, 131072, fake, 1, 8, fake, fake, fake, fake, fake, ws, n, 0, None)  # noqa: E731
    for ws, n in ((None, 0), (fake, need - 1), (fake + 16, need)):
        assert score(ws, n) == -1 and "workspace" in err()
    need = v.hip.vox_hip_linear_i8_workspace(0, 3, 100, 7, fake, 100)
    lin = lambda ws, n, ys=7: v.hip.vox_hip_linear_i8(0, fake, 100, 3, 100, 7, fake, 100, fake, None, fake, ys, ws, n, 0, None)  # noqa: E731
    assert need > 0 and lin(fake, need - 1) == -1 and "workspace" in err()
    assert lin(fake, need, 6) == -1 and "strides" in err()
    assert v.hip.vox_hip_linear_i8_workspace(0, 3, 131073, 7, fake, 131073) == -1 and "131072" in err()
    assert v.hip.vox_hip_linear_i8_workspace(0, 4194241, 64, 7, fake, 64) == -1 and "rows" in err()
    assert v.hip.vox_hip_linear_i8_workspace(0, 4194240, 64, 1 << 24, fake, 64) == -1 and "N" in err()
    assert v.hip.vox_hip_quantize_rows_i8(0, None, 8, 2, 8, fake, fake, 0, None) == -1 and "null" in err()
    far = 1 << 24                                                      # (a grid's threads are counted in 32 bits)
    assert v.hip.vox_hip_tree_plan(fake, None, far, 1, fake, fake, 0, None) == -1 and "batch" in err()
    assert v.hip.vox_hip_tree_accept(*[fake] * 7, far, 1, *[fake] * 4, 0, None) == -1 and "batch" in err()
    assert v.hip.vox_hip_tree_commit(0, 1, far, 1, 1, 8, 9, fake, st, fake, st, fake, st, fake, st, fake, fake, fake, 0, None) == -1 and "batch" in err()
    assert v.hip.vox_hip_token_scores_workspace(0, far, 1, 0) == -1 and "rows" in err()
    if v.device_count() == 0:
        assert v.hip.vox_hip_tree_plan(fake, None, 1, 4, fake, fake, 0, None) == -1 and "no such device" in err()


def test_compiled_calls_hand_back_what_they_do_not_take():
    """Tensors on the CPU, other things than tensors, wrong counts: None, so that the Python call says what is wrong."""
    c, x, t = ops._call, zeros(2, 16), zeros(2, 3, dtype=torch.int32)
    q = zeros(1, 2, 4, 16)
    for done in (c.tree_plan(t, None), c.tree_plan([1], None), c.tree_plan(t), c.tree_plan(t, 3), c.quantize_rows_i8(x), c.quantize_rows_i8(None), c.quantize_rows_i8(),
                 c.linear_i8(x, x, x, None), c.linear_i8(x, x.char(), x[0], 1.0), c.token_scores(x, None, 0), c.token_scores(x, None, 2 ** 80), c.token_scores(x, None, 1.5),
                 c.tree_accept(*[t] * 7), c.tree_commit(*[q[None]] * 4, t, t, t), c.tree_attention(*[q] * 8, None, 0, True), c.tree_attention(*[q] * 8, "1", None, 1)):
        assert done is None
    with pytest.raises(TypeError, match="arguments"):
        c.bind(print, 1)
