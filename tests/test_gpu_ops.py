"""GPU: the draft-verification operators (vox_hip_ops.h through voxtral_c_amd.ops) against their definitions in 64 bits.

Tolerances count roundings (half a step each: f32 2^-24, bf16 2^-8, f16 2^-11) and are worked out in ops_util.py or beside the check.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import ops_util as ref
from conftest import model_dir

import voxtral_c_amd as v
from voxtral_c_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16, I32 = torch.float32, torch.bfloat16, torch.float16, torch.int32


@pytest.fixture(autouse=True)
def need_gpu():
    if v.device_count() < 1:
        pytest.fail("no HIP device: the product has no CPU fallback")


def dev(a):
    return torch.as_tensor(np.ascontiguousarray(a)).to(DEV)


def randn(rng, *shape, dtype=F32, scale=1.0):
    return torch.as_tensor((rng.standard_normal(shape) * scale).astype(np.float32)).to(dtype).to(DEV)


# ---- trees -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,T", [(1, 1), (3, 2), (2, 63), (2, 64), (3, 65), (1, 200), (4, 256)])
def test_tree_plan(B, T):
    rng = np.random.default_rng(B * 1000 + T)
    parents, n = ref.random_tree(rng, B, T)
    if T > 4:
        parents[-1, T // 2], parents[-1, T // 3] = T - 1, -5          # no earlier node: these and what hangs behind them are cut off
        n[-1] = T
    sets, depth = ref.plan(parents, n)
    a, d = ops.tree_plan(dev(parents), dev(n))
    assert np.array_equal(d.cpu().numpy(), depth) and np.array_equal(a.cpu().numpy(), ref.words(sets, T))
    chain = np.arange(-1, T - 1, dtype=np.int32)[None]
    a, d = ops.tree_plan(dev(chain))
    assert np.array_equal(d.cpu().numpy()[0], np.arange(T)) and np.array_equal(a.cpu().numpy(), ref.words(ref.plan(chain, [T])[0], T))


def test_tree_plan_impossible_counts():
    parents = np.array([[-1, 0, 1]] * 3, np.int32)
    _, d = ops.tree_plan(dev(parents), dev(np.array([-7, 99, 1], np.int32)))
    assert d.cpu().tolist() == [[-1, -1, -1], [0, 1, 2], [0, -1, -1]]
    _, d = ops.tree_plan(dev(parents).repeat(1, 2)[:, ::2], None)      # a table that is not contiguous
    assert d.cpu().tolist() == [[0, -1, 1]] * 3                        # (parents -1, 1, 0: node 1's parent is itself, node 2's is node 0)


@pytest.mark.parametrize("B,T,kinds", [(1, 1, 2), (1, 2, 1), (5, 7, 2), (3, 64, 2), (2, 65, 3), (2, 256, 1)])
def test_tree_accept(B, T, kinds):
    rng = np.random.default_rng(T + kinds)
    for trial in range(3):
        parents, n = ref.random_tree(rng, B, T)
        if T == 256 and trial == 0:
            parents[0] = np.arange(-1, T - 1)                          # a chain that is accepted whole (one kind of token)
        tokens, choices = rng.integers(0, kinds, (2, B, T)).astype(np.int32)
        root, length = rng.integers(0, kinds, B).astype(np.int32), rng.integers(-3, 5000, B).astype(np.int32)
        a, d = ops.tree_plan(dev(parents), dev(n))
        got = ops.tree_accept(dev(tokens), dev(choices), dev(root), dev(parents), a, d, dev(length))
        for g, w in zip(got, ref.accept(parents, n, tokens, choices, root, length)):
            assert np.array_equal(g.cpu().numpy(), w)


@pytest.mark.parametrize("dtype,L,B,T,Hk,D,cap", [(F32, 2, 1, 2, 8, 128, 40), (BF16, 3, 3, 9, 2, 64, 9), (F16, 1, 2, 70, 3, 33, 100), (BF16, 2, 2, 5, 1, 4, 6)])
def test_tree_commit(dtype, L, B, T, Hk, D, cap):
    rng = np.random.default_rng(T * D)
    k, v_ = randn(rng, L, B, T, Hk, D, dtype=dtype), randn(rng, L, T, B, Hk, D, dtype=dtype).transpose(1, 2)
    kc, vc = randn(rng, L, B, cap, Hk, D, dtype=dtype), randn(rng, L, B, Hk, cap, D + 1, dtype=dtype)[..., 1:].transpose(2, 3)
    n = np.array([min(T, 1 + 7 * b) for b in range(B)], np.int32)
    path = np.full((B, T), -1, np.int32)
    for b in range(B):
        path[b, : n[b]] = np.sort(rng.permutation(T)[: n[b]])
    length = np.array([cap * 3 - 1 + b for b in range(B)], np.int32)
    wk, wv = kc.clone(), vc.clone()
    for b in range(B):
        for j in range(n[b]):
            slot = (int(length[b]) + j) % cap
            wk[:, b, slot], wv[:, b, slot] = k[:, b, path[b, j]], v_[:, b, path[b, j]]
    path[-1, n[-1]:] = T + 5                                           # behind the count: never read
    ops.tree_commit(k, v_, kc, vc, dev(path), dev(n), dev(length))
    assert torch.equal(kc, wk) and torch.equal(vc, wv)
    ops.tree_commit(k[0], v_[0], kc[0], vc[0], dev(path * 0 - 1), dev(n), dev(length))            # no node at all: nothing changes
    ops.tree_commit(k[0], v_[0], kc[0], vc[0], dev(path), dev(n * 0 - 4), dev(length))
    assert torch.equal(kc, wk) and torch.equal(vc, wv)


# ---- attention ---------------------------------------------------------------------------------------------------------------
def attn_case(seed, dtype, B, T, H, Hk, D, cap, lengths, shorter=True):
    rng = np.random.default_rng(seed)
    parents, n = ref.random_tree(rng, B, T, shorter)
    sets, depth = ref.plan(parents, n)
    f = lambda *s, scale=1.0: randn(rng, *s, dtype=dtype, scale=scale)  # noqa: E731
    return dict(q=f(B, T, H, D, scale=1.5), k=f(B, T, Hk, D), v=f(B, T, Hk, D), k_cache=f(B, cap, Hk, D), v_cache=f(B, cap, Hk, D),
                cache_len=dev(np.resize(np.array(lengths, np.int32), B)), ancestors=dev(ref.words(sets, T)), depth=dev(depth))


def check_attn(c, window=0, scale=None):
    D = c["q"].shape[3]
    out, lse = ops.tree_attention(**c, window=window, scale=scale, return_lse=True)
    w = ref.attention(c["q"], c["k"], c["v"], c["k_cache"], c["v_cache"], c["cache_len"].cpu().numpy(), c["ancestors"].cpu().numpy(), c["depth"].cpu().numpy(),
                      D ** -0.5 if scale is None else scale, window)
    off = np.abs(out.cpu().double().numpy() - w[0])
    assert np.isfinite(off).all() and (off <= ref.attention_bound(w[0], w[2], w[4], c["q"].dtype)).all(), float(off.max())
    got = lse.cpu().double().numpy()
    empty = np.isneginf(w[1])
    assert np.array_equal(np.isneginf(got), empty) and (np.abs(got[~empty] - w[1][~empty]) <= w[3][~empty]).all()
    return out, lse


ATTN = [
    # B, T, H, Hk, D, cap, lengths, window
    (1, 1, 4, 1, 128, 64, [0], 0), (1, 1, 8, 2, 128, 64, [1], 0), (2, 2, 32, 8, 128, 300, [232, 17], 8192),
    (3, 7, 4, 4, 64, 83, [200, 5, 83], 75), (2, 24, 8, 2, 128, 500, [499, 0], 0), (2, 64, 4, 1, 128, 200, [1000, 31], 150),
    (1, 65, 6, 2, 64, 100, [37], 0), (1, 256, 8, 2, 64, 40, [40], 9), (4, 5, 3, 3, 96, 70, [70, 69, 1, 33], 0), (1, 33, 8, 1, 128, 129, [128], 0),
    (2, 3, 4, 2, 256, 50, [49, 50], 0), (2, 3, 5, 5, 33, 20, [44, 7], 11), (1, 4, 4, 2, 1, 9, [9], 0), (1, 17, 12, 4, 80, 64, [64], 1), (1, 6, 16, 1, 192, 90, [77], 0),
    (2, 3, 8, 2, 128, 1500, [1500, 1111], 0), (1, 16, 4, 1, 64, 2100, [2099], 2000),
    (16, 12, 32, 8, 64, 1000, [1000, 612, 999], 0), (16, 24, 32, 8, 128, 700, [3000, 700, 350, 64], 600), (32, 2, 32, 16, 128, 900, [900, 31, 1800], 0),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", ATTN, ids=lambda c: "x".join(map(str, c[:6])))
def test_tree_attention(case, dtype):
    B, T, H, Hk, D, cap, lengths, window = case
    check_attn(attn_case(T * 7 + D, dtype, B, T, H, Hk, D, cap, lengths), window)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_strides(dtype):
    """Heads in front of rows, q;k;v side by side in one buffer, an offset of one element, a cache of which every other row is ours."""
    c = attn_case(3, dtype, 2, 5, 8, 2, 128, 60, [60, 21])
    plain = check_attn(c)
    merged = torch.cat([c["q"].flatten(2), c["k"].flatten(2), c["v"].flatten(2)], 2)
    q, k, v_ = (t.unflatten(2, (-1, 128)) for t in merged.split([1024, 256, 256], 2))
    kc = c["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)
    vc = torch.stack([c["v_cache"], torch.full_like(c["v_cache"], math.nan)], 2).flatten(1, 2)[:, ::2]
    got = check_attn({**c, "q": q, "k": k, "v": v_, "k_cache": kc, "v_cache": vc})
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
    odd = {n: torch.cat([c[n].flatten()[:1], c[n].flatten()])[1:].view(c[n].shape) for n in ("q", "k", "v", "k_cache", "v_cache")}
    check_attn({**c, **odd})
    one = c["k_cache"][:, :1].expand(2, 60, 2, 128)                    # broadcast inputs are read as they are
    check_attn({**c, "k_cache": one})


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("H", [4, 16, 24])
def test_tree_attention_ignores_what_is_masked(dtype, D, H):
    """NaN, infinities and the type's largest values in rows that nobody (or not everybody) may see."""
    B, T, window, cap = 2, 6, 20, 40
    c = attn_case(11, dtype, B, T, H, 2, D, cap, [33, 9])
    clean = check_attn(c, window)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dtype).max, torch.finfo(dtype).min):
        x = {**c, **{n: c[n].clone() for n in ("k", "v", "k_cache", "v_cache")}}
        x["k_cache"][0, :33 - window + 1], x["v_cache"][0, :33 - window + 1] = bad, bad       # in front of everybody's window
        x["k_cache"][0, 33:], x["v_cache"][0, 33:], x["k_cache"][1, 9:], x["v_cache"][1, 9:] = bad, bad, bad, bad
        got = ops.tree_attention(**x, window=window, return_lse=True)
        assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1]), bad
        # a node that only itself sees, and a cached row in front of the window of the deeper nodes
        x["k"][:, T - 1], x["v"][:, T - 1] = bad, bad
        x["k_cache"][0, 33 - window + 1], x["v_cache"][0, 33 - window + 1] = bad, bad
        got = ops.tree_attention(**x, window=window, return_lse=True)
        d = c["depth"].cpu().numpy()
        for b in range(B):
            for i in range(T - 1):
                sees = b == 0 and d[b, i] == 0
                if not sees:
                    assert torch.equal(got[0][b, i], clean[0][b, i]) and torch.equal(got[1][b, i], clean[1][b, i]), (bad, b, i)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_any_mask(dtype):
    """Masks that are no trees: rows of nothing, of everything, of one bit; bits behind the last node are not read."""
    c = attn_case(5, dtype, 2, 70, 4, 1, 128, 20, [0, 20], shorter=False)
    a = c["ancestors"].clone()
    a[:, 0], a[:, 1], a[:, 2, 0], a[:, 2, 1] = 0, -1, 0, 1 << 5
    c["ancestors"] = a
    out, lse = check_attn(c)
    assert (out[0, 0] == 0).all() and torch.isneginf(lse[0, 0]).all() and torch.isfinite(lse[1, 0]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("H", [2, 40])
def test_tree_attention_passes_on_what_is_seen(dtype, H):
    """An infinite value in the tree or at a window's edge reaches the rows that see it, with its sign, and nobody else; NaN and both signs give NaN."""
    window, D, T = 12, 64, 3
    c = attn_case(13, dtype, 1, T, H, 2, D, 16, [14], shorter=False)
    c["ancestors"] = dev(np.array([[[1], [3], [5]]], np.int64))        # nodes 1 and 2 hang behind node 0
    c["depth"] = dev(np.array([[0, 1, 1]], np.int32))
    clean = check_attn(c, window)[0]
    c["v"][0, 1, 0, 5], c["v"][0, 2, 1, 7] = math.inf, -math.inf
    c["v_cache"][0, 14 - window + 1, 0, 9] = -math.inf                 # seen by node 0 only
    c["v_cache"][0, 14 - window + 2, 1, 11], c["v"][0, 0, 1, 11] = math.inf, -math.inf          # both seen by all
    c["v_cache"][0, 13, 0, 3] = math.nan
    out = ops.tree_attention(**c, window=window).float().view(T, 2, H // 2, D)
    want = clean.float().view(T, 2, H // 2, D).clone()
    want[1, 0, :, 5], want[2, 1, :, 7], want[0, 0, :, 9], want[:, 1, :, 11], want[:, 0, :, 3] = math.inf, -math.inf, -math.inf, math.nan, math.nan
    assert torch.equal(torch.nan_to_num(out, nan=1e9, posinf=2e9, neginf=-2e9), torch.nan_to_num(want, nan=1e9, posinf=2e9, neginf=-2e9))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H", [2, 4, 40])
def test_tree_attention_depths_of_ones_own(dtype, H):
    """Depths that no tree of this size has (nodes far behind the cache's end): windows that lie inside, at the end of, and behind the cache."""
    c = attn_case(17, dtype, 2, 5, H, 2, 64, 300, [290, 120], shorter=False)
    c["depth"] = dev(np.array([[0, 150, 199, 200, 2 ** 31 - 1], [3, 60, 119, 1, -1]], np.int32))
    check_attn(c, window=200)
    check_attn(c, window=1)


def test_tree_attention_scale():
    c = attn_case(14, F32, 1, 5, 4, 2, 64, 40, [33])
    check_attn(c, scale=-0.2)
    check_attn(c, scale=1.5)
    d = attn_case(14, BF16, 2, 40, 4, 2, 128, 40, [33])
    check_attn(d, scale=-0.2)
    for bad in (0.0, math.inf, math.nan):
        with pytest.raises((v.VoxError, ValueError), match="scale"):
            ops.tree_attention(**c, scale=bad)


def test_tree_attention_scores_of_minus_infinity_and_nan():
    """A key of -inf scores: no weight; a row of nothing else is an empty row; a NaN that is seen makes its row NaN."""
    c = attn_case(6, F32, 1, 3, 2, 2, 64, 8, [4], shorter=False)
    c["q"].abs_()
    c["k_cache"][0, 1] = -math.inf
    keep = {n: t.clone() for n, t in c.items()}
    got = ops.tree_attention(**c)
    keep["cache_len"][:] = 3
    keep["k_cache"][0, 1:3], keep["v_cache"][0, 1:3] = c["k_cache"][0, 2:4], c["v_cache"][0, 2:4]
    want = ops.tree_attention(**keep)
    assert torch.allclose(got, want, rtol=0, atol=8 * 2.0 ** -24 * 5)   # the same weights in another order: sums of at most 7 terms of at most 5
    c["k_cache"][:], c["k"][:] = -math.inf, -math.inf
    out, lse = ops.tree_attention(**c, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    c["k"][0, 0, 0] = math.nan
    out = ops.tree_attention(**c)
    assert torch.isnan(out[0, 0, 0]).all() and (out[0, :, 1] == 0).all()


def test_tree_attention_nothing():
    c = attn_case(7, F32, 2, 3, 4, 2, 64, 8, [3, 4])
    assert ops.tree_attention(**{n: t[:0] for n, t in c.items()}).shape == (0, 3, 4, 64)
    e = {n: (t if "cache" in n else t[:, :0]) for n, t in c.items()}
    assert ops.tree_attention(**{**e, "ancestors": c["ancestors"][:, :0, :0]}).shape == (2, 0, 4, 64)
    c["cache_len"][:] = -9                                             # an empty cache
    check_attn(c)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_far_rows(dtype):
    """A cache whose rows lie more than 2^31 elements apart: offsets are 64 bits wide."""
    c = attn_case(8, dtype, 2, 2, 2, 1, 128, 6, [6, 5])
    far = torch.empty(2 ** 31 + 4096, dtype=dtype, device=DEV)
    near = {}
    for n in ("k_cache", "v_cache"):
        view = far.as_strided((2, 6, 1, 128), (2 ** 31, 256, 128, 1), 2048 if n == "v_cache" else 0)
        view.copy_(c[n])
        near[n] = view
    want = ops.tree_attention(**c)
    assert torch.equal(ops.tree_attention(**{**c, **near}), want)


# ---- scores ------------------------------------------------------------------------------------------------------------------
def scores_ref(x, tokens, top):
    x = x.detach().cpu().double().numpy()
    V = x.shape[1]
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(1, keepdims=True)
        lse = np.where(np.isneginf(m), -np.inf, m + np.log(np.exp(x - np.where(np.isneginf(m), 0, m)).sum(1, keepdims=True)))
        lp = np.where(np.isneginf(x), -np.inf, x - lse)
        entropy = -np.where(np.isneginf(lp), 0, np.exp(lp) * np.where(np.isneginf(lp), 0, lp)).sum(1)
    ids = tokens.cpu().numpy()
    inside = (ids >= 0) & (ids < V)
    given = np.where(inside, np.take_along_axis(lp, np.where(inside, ids, 0), 1), -np.inf)
    index = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return given, entropy, lse[:, 0], index, np.take_along_axis(lp, index, 1)


def check_scores(x, tokens, top):
    g = ops.token_scores(x, tokens, top)
    lp, entropy, lse, index, top_lp = scores_ref(x, tokens, top)
    V, e = x.shape[1], 2.0 ** -24
    fin = x.float().cpu().numpy()
    fin = fin[np.isfinite(fin)]
    span = float(fin.max() - fin.min()) if fin.size else 0.0
    # A term's exponent is off by 2 e of its size (at most the row's span, beyond which terms below e^-17 do not matter: 2 e * 17 + 2 e in all), the
    # sum by its depth: V / 1024 terms one after another per thread at least 4 times over, then joins.  log1p, the maximum's addition and x - lse: 3 e of
    # their sizes.
    sum_off = (2 * 17 + 4 + V / 64 + 64) * e
    size = np.abs(np.where(np.isfinite(lse), lse, 0)) + span
    def near(got, want, tol):
        got = got.cpu().double().numpy()
        same = np.isneginf(got) & np.isneginf(want)
        assert np.array_equal(np.isneginf(got), np.isneginf(want)) and (np.abs(np.where(same, 0, got) - np.where(same, 0, want)) <= tol).all(), np.abs(got - want)[~same].max()
    near(g.lse, lse, sum_off + 3 * e * size)
    near(g.logprob, lp, (sum_off + 3 * e * size)[:, None])
    near(g.top_logprob, top_lp, (sum_off + 3 * e * size)[:, None])
    near(g.entropy, entropy, sum_off * (2 + entropy) * 2 + 3 * e * size)
    assert np.array_equal(g.top_index.cpu().numpy(), index)
    return g


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,V,given,top", [(1, 1, 1, 1), (3, 2, 2, 2), (2, 63, 1, 5), (5, 1000, 3, 64), (1, 131072, 1, 8), (7, 50257, 2, 4), (40, 4097, 1, 0), (700, 257, 1, 1)])
def test_token_scores(dtype, R, V, given, top):
    rng = np.random.default_rng(V + R)
    x = randn(rng, R, V, dtype=dtype, scale=3.0)
    x[0, rng.integers(V)] = 25
    check_scores(x, dev(rng.integers(0, V, (R, given)).astype(np.int32)), top)


def test_token_scores_ties_zeros_and_order():
    """Equal logits by the lowest index, -0 equal to 0, rising and falling rows (every element new to the list, or none), odd strides."""
    V = 3001
    x = torch.zeros(6, V, device=DEV)
    x[0, ::3] = -0.0
    x[1] = torch.arange(V, device=DEV) * 0.01
    x[2] = -torch.arange(V, device=DEV) * 0.01
    x[3] = (torch.arange(V, device=DEV) % 7).float()
    x[4] = (torch.arange(V, device=DEV) // 500 % 2).float()
    x[5, 1234], x[5, 77] = 3, 3
    t = torch.zeros(6, 1, dtype=I32, device=DEV)
    for dtype in (F32, BF16, F16):
        check_scores(x.to(dtype), t, 64)
    big = torch.full((6, V + 7), math.nan, device=DEV)
    big[:, 3: 3 + V] = x
    g, w = ops.token_scores(big[:, 3: 3 + V], t, 9), ops.token_scores(x, t, 9)
    assert torch.equal(g.top_index, w.top_index)
    check_scores(big[:, 3: 3 + V], t, 9)
    check_scores(x[:1].expand(4, V), t[:4], 3)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("top", [1, 7, 64])
def test_token_scores_hard_orders(dtype, top):
    """Long rows that rise (every trip brings a new list), fall, are equal throughout, take few values, or hold their largest elements at one end."""
    V, rng = 40003, np.random.default_rng(top)
    at = np.arange(V, dtype=np.float32)
    x = np.stack([at * 1e-3, -at * 1e-3, np.full(V, 2.5), rng.integers(0, 3, V), rng.standard_normal(V), rng.standard_normal(V)]).astype(np.float32)
    x[4, -70:] += 30
    x[5, :70] += 30
    check_scores(dev(x).to(dtype), dev(np.array([[0], [1], [2], [3], [V - 1], [5]], np.int32)), top)


def test_token_scores_switched_off_and_broken_rows():
    V = 5000
    rng = np.random.default_rng(9)
    x = randn(rng, 6, V)
    x[0, 10:] = -math.inf                                              # ten tokens left, a list of twelve
    x[1] = -math.inf
    x[2] = -math.inf
    x[2, 4321] = -5.0                                                  # one token left
    t = dev(np.array([[0, 11], [5, -1], [4321, 4320], [3, V], [7, -2 ** 31], [1, 2 ** 31 - 1]], np.int32))
    g = check_scores(x, t, 12)
    assert g.top_index[0].tolist()[10:] == [10, 11] and g.entropy[2] == 0 and g.logprob[2, 0] == 0
    x[3, 17], x[4, 99], x[5, 3] = math.nan, math.inf, -math.nan
    g = ops.token_scores(x, t, 12)
    assert torch.isnan(g.lse[[3, 5]]).all() and torch.isnan(g.entropy[[3, 5]]).all() and torch.isnan(g.logprob[3]).all() and torch.isnan(g.top_logprob[3]).all()
    assert g.lse[4] == math.inf and torch.isnan(g.entropy[4]) and torch.isnan(g.logprob[4, 0])
    assert g.top_index[3, 0] == 17 and g.top_index[4, 0] == 99 and g.top_index[5, 0] == 3
    check_scores(x[:3], t[:3], 12)                                     # their neighbours are as before


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [70, 9001, 131072])
def test_token_scores_infinity_and_nan_in_one_row(dtype, V):
    """A NaN makes its row NaN wherever an infinity stands; without one, the infinity is the log-sum."""
    rng = np.random.default_rng(33)
    x = randn(rng, 9, V)
    x[:, 5] = math.inf
    at = [0, 4, 6, 33, V // 2, V - 1]
    for row, i in enumerate(at):
        x[row, i] = math.nan
    x[6, V - 2] = math.inf
    x[7, 6] = -math.inf
    for top in (0, 3):
        g = ops.token_scores(x.to(dtype), dev(np.full((9, 1), 7, np.int32)), top)
        assert torch.isnan(g.lse[:6]).all() and (g.lse[6:] == math.inf).all()
        assert torch.isnan(g.entropy).all() and torch.isnan(g.logprob).all()
        if top:
            assert g.top_index[:6, 0].tolist() == at and (g.top_index[:6, 1] == 5).all() and (g.top_index[6:, 0] == 5).all() and g.top_index[6, 1] == V - 2


def test_token_scores_confident_rows_keep_their_digits():
    """One token with almost all the probability: entropy and logprob are small numbers with all their digits, not differences of large ones."""
    x = torch.full((4, 4096), 0.0, device=DEV)
    for i, top in enumerate((12.0, 20.0, 30.0, 40.0)):
        x[i, 100 + i] = top
    t = dev(np.arange(100, 104, dtype=np.int32))
    g = ops.token_scores(x, t, 1)
    lp, entropy, _, _, _ = scores_ref(x, t[:, None], 1)
    assert g.logprob.shape == (4,)
    # relative: the sum of 4095 equal terms (exponent off by 2 e * 40, depth of the sum 64), log1p and the entropy's quotient
    tol = (2 * 40 + 4 + 64 + 64) * 2.0 ** -24
    s = 4095 * np.exp(-np.array([12.0, 20.0, 30.0, 40.0]))
    exact_lp, exact_h = -np.log1p(s), np.log1p(s) + s / (1 + s) * np.array([12.0, 20.0, 30.0, 40.0])
    assert (np.abs(g.logprob.cpu().double().numpy() / exact_lp - 1) <= tol).all() and (np.abs(g.entropy.cpu().double().numpy() / exact_h - 1) <= 2 * tol).all()


def test_token_scores_nothing():
    g = ops.token_scores(torch.zeros(0, 10, device=DEV), None, 3)
    assert g.logprob.shape == (0, 0) and g.entropy.shape == (0,) and g.top_index.shape == (0, 3)
    g = ops.token_scores(torch.zeros(2, 10, device=DEV))
    assert g.logprob.shape == (2, 0) and g.top_index.shape == (2, 0) and (g.lse.cpu() - math.log(10)).abs().max() <= 4 * 2.0 ** -24 * math.log(10)


# ---- 8-bit integers ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,K", [(1, 1), (3, 64), (2, 1000), (5, 4099), (300, 128), (2, 4096), (3, 4100), (2, 8192), (2, 8200), (1, 20000)])
def test_quantize_rows(dtype, R, K):
    rng = np.random.default_rng(R * K)
    x = randn(rng, R, K, dtype=dtype, scale=10.0)
    q, s = ops.quantize_rows_i8(x)
    wq, ws = ref.quantize(x)
    assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws)


def test_quantize_rows_borders():
    """Quotients on and next to the half numbers, rows of zeros, of subnormal numbers, of the largest ones, and broken rows."""
    rng = np.random.default_rng(1)
    rows = []
    for amax in (127.0, 1.0, 0.3, 3.3e38, 1e-30, 2.0 ** -126, 1e-40, 1e-45):
        s = np.maximum(np.float32(amax) / np.float32(127), np.float32(2.0 ** -126))
        half = ((np.arange(-127, 127) + 0.5) * np.float64(s)).astype(np.float32)
        half = np.clip(half, -np.float32(amax), np.float32(amax))
        rows.append(np.concatenate([[np.float32(amax)], half, np.nextafter(half, np.float32(np.inf)), np.nextafter(half, np.float32(-np.inf))]).astype(np.float32))
    x = np.clip(np.stack(rows), -np.abs(np.stack(rows)[:, :1]), np.abs(np.stack(rows)[:, :1]))
    x = np.concatenate([x, np.zeros((3, x.shape[1]), np.float32)])
    x[-2, 5], x[-1, 7] = np.inf, np.nan
    q, s = ops.quantize_rows_i8(dev(x))
    wq, ws = ref.quantize(torch.as_tensor(x))
    assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws, equal_nan=True)


def check_linear(x, w, ws, bias, dtype):
    y = ops.linear_i8(x, w, ws, bias)
    q, s = ref.quantize(x)
    # whole numbers below 2^31: their product in float64 is exact
    exact = (q.astype(np.float64) @ w.cpu().numpy().astype(np.float64).T) * s[:, None].astype(np.float64) * ws.cpu().double().numpy()
    b = 0 if bias is None else bias.detach().cpu().double().numpy()
    # the sum's conversion, two products and the bias in f32, then the storage rounding
    tol = 2.0 ** -24 * (4 * np.abs(exact) + np.abs(exact + b)) + (ref.HALF[dtype] * 1.01 * np.abs(exact + b) if dtype != F32 else 0) + 1e-37
    if dtype == F16:
        tol = tol + 2.0 ** -25                                         # numbers below f16's normal ones
    off = np.abs(y.cpu().double().numpy() - (exact + b))
    assert y.dtype == dtype and (off <= tol).all(), (off - tol).max()
    return y


I8 = [(1, 64, 16), (1, 1280, 6144), (2, 100, 7), (3, 1, 5), (5, 128, 1000), (16, 256, 48), (17, 320, 130), (25, 5120, 1280), (33, 80, 64), (64, 4096, 33), (65, 1008, 257), (130, 192, 96),
      (200, 1280, 520), (257, 2064, 129), (1000, 64, 65), (300, 77, 200), (128, 128, 128), (256, 512, 256), (513, 640, 768),
      (700, 144, 5500), (1030, 208, 8000), (33, 2048, 300), (64, 5120, 1280), (70, 1536, 2000), (129, 4096, 1000), (40, 640, 127), (16, 1024, 100), (4, 4096, 65), (13, 1248, 96), (1, 16384, 40)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,K,N", I8)
def test_linear_i8(dtype, M, K, N):
    rng = np.random.default_rng(M * N + K)
    x = randn(rng, M, K, dtype=dtype, scale=2.0)
    w = dev(rng.integers(-128, 128, (N, K)).astype(np.int8))
    ws = dev((rng.random(N).astype(np.float32) + 0.1) / (127 * math.sqrt(K)))
    check_linear(x, w, ws, randn(rng, N, dtype=dtype) if N % 2 else None, dtype)


def test_linear_i8_largest_sums():
    """Every product of the same sign and size at the largest K: sums next to 2^31."""
    K = 131072
    x, w = torch.full((2, K), -3.0, device=DEV), torch.full((3, K), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    check_linear(x, w, torch.ones(3, device=DEV), None, F32)


def test_linear_i8_strides_and_broken_rows():
    rng = np.random.default_rng(4)
    for M in (1, 7, 40, 200):
        x, w = randn(rng, M, 3 * 256)[:, 256:512], dev(rng.integers(-127, 128, (90, 300)).astype(np.int8))
        ws = torch.rand(90, device=DEV) / 1000
        a = check_linear(x, w[:, :256], ws, None, F32)                 # rows of 300 bytes: not a multiple of 16
        b = check_linear(x, w[:, :256].contiguous(), ws, None, F32)
        c = check_linear(x, w[:, 3:259], ws, None, F32)                # off by three bytes
        assert torch.equal(a, b) and not torch.equal(a, c)
        d = check_linear(x[:1].expand(M, 256), w[:1, :256].expand(90, 256), ws, None, F32)
        assert (d == d[:1]).all()
        bad = x.clone()
        bad[0, 3] = math.nan
        y = ops.linear_i8(bad, w[:, :256], ws)
        assert torch.isnan(y[0]).all() and torch.equal(y[1:], a[1:])
        bad[0, 3] = -math.inf
        assert torch.isnan(ops.linear_i8(bad, w[:, :256], ws)[0]).all()
    x[0] = 0
    assert (ops.linear_i8(x, w[:, :256], ws, torch.arange(90.0, device=DEV))[0].cpu() == torch.arange(90.0)).all()


def test_linear_i8_nothing():
    w, ws = torch.zeros(5, 64, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV)
    assert ops.linear_i8(torch.zeros(0, 64, device=DEV), w, ws).shape == (0, 5)
    assert ops.linear_i8(torch.zeros(3, 64, device=DEV), w[:0], ws[:0]).shape == (3, 0)
    assert ops.quantize_rows_i8(torch.zeros(0, 64, device=DEV))[0].shape == (0, 64)


# ---- together ----------------------------------------------------------------------------------------------------------------
class Tiny:
    """A decoder of two layers whose products run in 8 bits: attention block, feed-forward block, logits of the tied embedding."""

    H, Hk, D, X, F, V, L = 4, 2, 64, 128, 192, 500, 2

    def __init__(self, seed, dtype):
        rng = np.random.default_rng(seed)
        w8 = lambda n, k: ops.quantize_rows_i8(randn(rng, n, k, scale=1.0 / math.sqrt(k)))  # noqa: E731
        qkv = (self.H + 2 * self.Hk) * self.D
        self.layers = [dict(qkv=w8(qkv, self.X), wo=w8(self.X, self.H * self.D), up=w8(self.F, self.X), down=w8(self.X, self.F)) for _ in range(self.L)]
        self.emb, self.pos, self.dtype = randn(rng, self.V, self.X, scale=1.5), randn(rng, 400, self.X), dtype
        self.head = ops.quantize_rows_i8(self.emb)

    def rows(self, tokens, positions, k_cache, v_cache, cache_len, ancestors, depth):
        """tokens, positions [B, T] -> logits [B * T, V] and every layer's keys and values of the rows."""
        B, T = tokens.shape
        x, ks, vs = (self.emb[tokens.long()] + self.pos[positions.long()]).view(B * T, self.X), [], []
        for l, w in enumerate(self.layers):
            norm = lambda y: (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5)).to(self.dtype)  # noqa: E731
            q, k, v_ = ops.linear_i8(norm(x), *w["qkv"]).view(B, T, -1, self.D).split([self.H, self.Hk, self.Hk], 2)
            ks.append(k), vs.append(v_)
            o = ops.tree_attention(q, k, v_, k_cache[l], v_cache[l], cache_len, ancestors, depth)
            x = x + ops.linear_i8(o.view(B * T, -1), *w["wo"]).float()
            x = x + ops.linear_i8(torch.relu(ops.linear_i8(norm(x), *w["up"])), *w["down"]).float()
        return ops.linear_i8(norm(x).float(), *self.head), torch.stack(ks), torch.stack(vs)


def decode_step_by_step(m, prompt, steps, cap):
    """One token at a time: the cache's rows, the choices."""
    B = prompt.shape[0]
    kc, vc = (torch.zeros(m.L, B, cap, m.Hk, m.D, dtype=m.dtype, device=DEV) for _ in range(2))
    a, d = ops.tree_plan(torch.full((B, 1), -1, dtype=I32, device=DEV))
    token, out = prompt[:, 0], []
    for i in range(prompt.shape[1] + steps):
        n = torch.full((B,), i, dtype=I32, device=DEV)
        logits, k, v_ = m.rows(token[:, None], n[:, None], kc, vc, n, a, d)
        ops.tree_commit(k, v_, kc, vc, torch.zeros(B, 1, dtype=I32, device=DEV), torch.ones(B, dtype=I32, device=DEV), n)
        choice = ops.token_scores(logits, top=1).top_index[:, 0]
        token = prompt[:, i + 1] if i + 1 < prompt.shape[1] else choice
        if i + 1 >= prompt.shape[1]:
            out.append(choice)
    return torch.stack(out, 1).cpu().numpy()


def test_verification_passes_give_the_ids_of_single_steps():
    """Greedy decoding through draft trees (right drafts, wrong ones, siblings) gives exactly the ids of one token at a time.  In f32: the products of
    whole numbers are exact and the attention's sums differ in their last bits only, far below the margins of these logits."""
    m, cap, steps, B = Tiny(3, F32), 64, 40, 2
    rng = np.random.default_rng(8)
    prompt = dev(rng.integers(0, m.V, (B, 3)).astype(np.int32))
    want = decode_step_by_step(m, prompt, steps + 8, cap)
    kc, vc = (torch.zeros(m.L, B, cap, m.Hk, m.D, dtype=m.dtype, device=DEV) for _ in range(2))
    cache_len, root = torch.zeros(B, dtype=I32, device=DEV), prompt[:, 0].clone()
    got, passes = [prompt[b, :1].tolist() for b in range(B)], 0
    while min(map(len, got)) < steps and passes < 3 * steps:
        # node 0: the token that is known; behind it two siblings, a chain of three behind the second one; drafts are right three times in four
        full = [prompt[b].tolist() + want[b].tolist() for b in range(B)]
        known = [len(g) for g in got]
        draft = np.zeros((B, 6), np.int32)
        parents = np.array([[-1, 0, 0, 2, 3, 4]] * B, np.int32)
        for b in range(B):
            nxt = (full[b] + [0] * 8)[known[b] - 1: known[b] + 5]
            draft[b] = [nxt[0], (nxt[1] + 1) % m.V, nxt[1], nxt[2], nxt[3], nxt[4]]
            if rng.random() < 0.25:
                draft[b, 1 + rng.integers(5)] = rng.integers(m.V)
        tok, par = dev(draft), dev(parents)
        a, d = ops.tree_plan(par)
        logits, k, v_ = m.rows(tok, cache_len[:, None] + d, kc, vc, cache_len, a, d)
        choices = ops.token_scores(logits, top=1).top_index.view(B, 6)
        forced = choices.clone()
        for b in range(B):                                             # inside the prompt the next token is given
            for i, dep in enumerate([0, 1, 1, 2, 3, 4]):
                if known[b] + dep < prompt.shape[1]:
                    forced[b, i] = prompt[b, known[b] + dep]
        path, n, after, new_len = ops.tree_accept(tok, forced, root, par, a, d, cache_len)
        ops.tree_commit(k, v_, kc, vc, path, n, cache_len)
        for b in range(B):
            got[b] += [int(t) for t in draft[b][path[b, 1: n[b]].cpu().numpy()]] + [int(after[b])]
        cache_len, root, passes = new_len, after, passes + 1
    for b in range(B):
        ids = (prompt[b].tolist() + want[b].tolist())[: steps]
        assert got[b][: steps] == ids
    assert passes < steps                                              # several ids per pass


def captured_state(seed, dtype=BF16):
    c = attn_case(seed, dtype, 2, 9, 8, 2, 128, 300, [290, 100], shorter=False)
    rng = np.random.default_rng(seed)
    parents, _ = ref.random_tree(rng, 2, 9, False)
    c.update(parents=dev(parents), logits=randn(rng, 18, 20000, dtype=dtype), x=randn(rng, 18, 512, dtype=dtype), w=dev(rng.integers(-127, 128, (640, 512)).astype(np.int8)),
             ws=torch.rand(640, device=DEV) / 1000, root=dev(rng.integers(0, 3, 2).astype(np.int32)), tokens=dev(rng.integers(0, 3, (2, 9)).astype(np.int32)))
    return c


def verification_pass(c):
    a, d = ops.tree_plan(c["parents"])
    y = ops.linear_i8(c["x"], c["w"], c["ws"])
    o, lse = ops.tree_attention(c["q"], c["k"], c["v"], c["k_cache"], c["v_cache"], c["cache_len"], a, d, window=250, return_lse=True)
    s = ops.token_scores(c["logits"], c["tokens"].view(-1), 3)
    choices = (s.top_index[:, 0] % 3).view(2, 9)
    path, n, after, new_len = ops.tree_accept(c["tokens"], choices.contiguous(), c["root"], c["parents"], a, d, c["cache_len"])
    kc, vc = c["k_cache"].clone(), c["v_cache"].clone()
    ops.tree_commit(c["k"], c["v"], kc, vc, path, n, c["cache_len"])
    return [a, d, y, o, lse, *s, path, n, after, new_len, kc, vc]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_passes_replay():
    """Two graphs of a whole pass, replayed in turn on new inputs with eager work in between: every replay gives the eager result's bits."""
    one, two = captured_state(1), captured_state(2)
    for c in (one, two):
        verification_pass(c)
    torch.cuda.synchronize()
    graphs = []
    for c in (one, two):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = verification_pass(c)
        graphs.append((g, r, c))
    for trial in range(4):
        for n, (g, r, c) in enumerate(graphs):
            fresh = captured_state(10 * trial + n)
            for k in c:
                c[k].copy_(fresh[k])
        for g, _, _ in graphs:
            g.replay()
        wants = [verification_pass(c) for _, _, c in graphs]
        torch.cuda.synchronize()
        for (g, r, c), w in zip(graphs, wants):
            assert same(r, w), trial
            g.replay()
        torch.cuda.synchronize()
        for (g, r, c), w in zip(graphs, wants):
            assert same(r, w), trial


def test_two_streams_at_once():
    """Passes on two streams, and tensors made on another stream than the one that uses them (ordered by the caller): the single stream's bits."""
    states = [captured_state(s) for s in (21, 22)]
    wants = [verification_pass(c) for c in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [[], []]
    for _ in range(5):
        for i, (s, c) in enumerate(zip(streams, states)):
            with torch.cuda.stream(s):
                got[i].append(verification_pass(c))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(same(r, wants[i]) for r in got[i])


def test_results_do_not_change_from_call_to_call():
    for dtype in (F32, F16):
        c = captured_state(31, dtype)
        first = verification_pass(c)
        for _ in range(3):
            assert same(first, verification_pass(c))


def test_attention_over_the_engines_own_ring():
    """The C entry on an engine's decoder ring and stream: what vox_hip_decoder_kv_devptr gives is the operator's cache."""
    from audio_util import synth_speech
    with v.Model(model_dir("tiny"), enc_window=48, dec_window=64) as m:
        m.transcribe(synth_speech(5.0, 31))
        e, dims = m.engine, m.dims
        H, Hk, D, T = dims.dec_heads, dims.dec_kv_heads, dims.dec_head_dim, 4
        kp, vp, cap, n = C.c_void_p(), C.c_void_p(), C.c_int(), v.hip.vox_hip_decoder_kv_len(C.c_void_p(e))
        v.hip.vox_hip_decoder_kv_devptr.argtypes = [C.c_void_p, C.c_int, C.POINTER(C.c_void_p), C.POINTER(C.c_void_p), C.POINTER(C.c_int)]
        assert v.hip.vox_hip_decoder_kv_devptr(e, dims.dec_layers, C.byref(kp), C.byref(vp), C.byref(cap)) == -1
        assert v.hip.vox_hip_decoder_kv_devptr(e, 1, C.byref(kp), C.byref(vp), C.byref(cap)) == 0 and cap.value >= 64 and n > 10
        host = [np.empty((1, cap.value, Hk, D), np.float32) for _ in range(2)]
        v.hip.vox_hip_memcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
        for h, p in zip(host, (kp, vp)):
            assert v.hip.vox_hip_memcpy(e, h.ctypes.data, p.value, h.nbytes, 1) == 0
        c = attn_case(2, F32, 1, T, H, Hk, D, cap.value, [n], shorter=False)
        out, lse = torch.empty(1, T, H, D, device=DEV), torch.empty(1, T, H, device=DEV)
        st = lambda t: t.stride()[:3]  # noqa: E731
        args = ops._ATTN.pack(c["q"].data_ptr(), c["k"].data_ptr(), c["v"].data_ptr(), kp.value, vp.value, c["cache_len"].data_ptr(), c["ancestors"].data_ptr(),
                              c["depth"].data_ptr(), out.data_ptr(), lse.data_ptr(), *st(c["q"]), *st(c["k"]), *st(c["v"]), *st(c["k_cache"]), *st(c["v_cache"]), *st(out),
                              0, 1, T, H, Hk, D, cap.value, dims.dec_window, D ** -0.5, 0)
        need = v.hip.vox_hip_tree_attention_workspace(args)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
        v.hip.vox_hip_stream_handle.restype = C.c_void_p
        v.hip.vox_hip_stream_handle.argtypes = [C.c_void_p]
        torch.cuda.synchronize()
        assert v.hip.vox_hip_tree_attention(args, ws.data_ptr(), need, 0, v.hip.vox_hip_stream_handle(e)) == 0
        v.hip.vox_hip_sync(e)
        w = ref.attention(c["q"], c["k"], c["v"], torch.as_tensor(host[0]), torch.as_tensor(host[1]), [n], c["ancestors"].cpu().numpy(), c["depth"].cpu().numpy(), D ** -0.5, dims.dec_window)
        assert (np.abs(out.cpu().double().numpy() - w[0]) <= ref.attention_bound(w[0], w[2], w[4], F32)).all() and (np.abs(lse.cpu().double().numpy() - w[1]) <= w[3]).all()


class HandsBack:
    def __getattr__(self, name):
        return lambda *args: None


def test_compiled_calls_and_their_python_twins_agree(monkeypatch):
    """What the compiled calls take and what they hand back run the same kernels: equal bits, and ordinary arguments are taken."""
    for dtype in (F32, BF16, F16):
        c = captured_state(41, dtype)
        want = verification_pass(c)
        assert ops._call.quantize_rows_i8(randn(np.random.default_rng(1), 3, 40, dtype=dtype)) is not None
        with monkeypatch.context() as m:
            m.setattr(ops, "_call", HandsBack())
            assert same(want, verification_pass(c))


def test_wrong_calls_on_the_gpu_are_refused():
    rng = np.random.default_rng(3)
    q, k, kc = randn(rng, 2, 3, 4, 16), randn(rng, 2, 3, 2, 16), randn(rng, 2, 9, 2, 16)
    length = dev(np.array([4, 20], np.int32))
    words, depth = ops.tree_plan(dev(np.array([[-1, 0, 1], [-1, -1, 0]], np.int32)))
    good = [q, k, k.clone(), kc, kc.clone(), length, words, depth]
    out = ops.tree_attention(*good)
    assert torch.equal(out, ops.tree_attention(*good, scale=16 ** -0.5, window=0)) and torch.equal(out, ops.tree_attention(*good, window=2 ** 40))
    for i, bad in ((0, q.half()), (0, q[:, :, :3]), (0, q.cpu()), (1, k[:1]), (2, k.double()), (3, kc[..., :8]), (4, kc.transpose(2, 3)), (5, length.long()), (5, length[:1]),
                   (6, words.int()), (7, depth[:, :2]), (7, depth.cpu()), (1, k.clone().requires_grad_())):
        with pytest.raises(ValueError, match="tree_attention"):
            ops.tree_attention(*good[:i], bad, *good[i + 1:])
    for scale in (0.0, math.inf, math.nan):
        with pytest.raises(v.VoxError, match="scale"):
            ops.tree_attention(*good, scale=scale)
    spread = torch.stack([depth, depth], 2)[:, :, 0]                   # a table that is not contiguous is copied
    assert torch.equal(out, ops.tree_attention(*good[:7], spread))
    x, w, s = randn(rng, 3, 32), torch.ones(5, 32, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda")
    assert ops.linear_i8(x, w, s).shape == (3, 5)
    for args in ((x, w[:, :16], s), (x, w, s[:4]), (x, w.float(), s), (x, w, s, s[:2]), (x, w, s, s.half()), (x, w, s.cpu()), (x, w, s.clone().requires_grad_()), (x.double(), w, s)):
        with pytest.raises(ValueError, match="linear_i8"):
            ops.linear_i8(*args)
    for args in ((x, None, 33), (x, None, -1), (x, dev(np.zeros((2, 1), np.int32))), (x, dev(np.zeros((3, 1), np.int64))), (x[0],), (x.t(),)):
        with pytest.raises(ValueError, match="token_scores"):
            ops.token_scores(*args)
    t = dev(np.zeros((2, 3), np.int32))
    with pytest.raises(ValueError, match="tree_accept"):
        ops.tree_accept(t, t, length, t, words, depth[:1], length)
    n = dev(np.ones(2, np.int32))
    for a in ((k, k, kc[:, :2], kc[:, :2]), (k, k, kc[:, :1].expand(2, 9, 2, 16), kc), (k, k, kc.half(), kc), (k, k.cpu(), kc, kc)):
        with pytest.raises(ValueError, match="tree_commit"):
            ops.tree_commit(*a, t, n, length)
