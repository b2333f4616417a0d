"""GPU: calls of the draft-verification operators at the edges of what their definitions allow, against 64 bits (test_gpu_ops.py has the ordinary ones)."""
import math

import numpy as np
import pytest
import torch

from test_gpu_ops import attn_case, check_linear

import voxtral_c_amd as v
from voxtral_c_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16, I32 = torch.float32, torch.bfloat16, torch.float16, torch.int32


@pytest.fixture(autouse=True)
def need_gpu():
    if v.device_count() < 1:
        pytest.fail("no HIP device: the product has no CPU fallback")


# ---- scores: tokens switched off with the type's lowest number -----------------------------------------------------------------
def check_switched_off(x, live, tokens, top):
    """x [rows, V], live [V] truth values: the tokens that are not switched off.  The tolerances are those of ordinary rows, from the live tokens' span."""
    g = ops.token_scores(x, tokens, top)
    assert not any(torch.isnan(t).any() for t in (g.logprob, g.entropy, g.lse, g.top_logprob))
    x64 = x.cpu().double().numpy()
    m = x64.max(1, keepdims=True)
    log1 = np.log(np.exp(x64 - m).sum(1, keepdims=True))               # (apart from m, next to which it may be nothing)
    lse, lp = (m + log1)[:, 0], (x64 - m) - log1
    p = np.exp(lp)
    entropy = -np.where(p > 0, p * lp, 0).sum(1)
    index = np.argsort(-x64, axis=1, kind="stable")[:, :top]
    V, e = x.shape[1], 2.0 ** -24
    size = log1 + (np.ptp(x64[:, live]) if live.any() else 0.0)
    # Exponents are off by 2 e of their size (17 at most, smaller terms do not matter), sums by their depth; the maximum's addition, x - max and log1p
    # by 3 e of their sizes.
    sum_off = (2 * 17 + 4 + V / 64 + 64) * e

    def near(got, want, tol):
        off = np.abs(got.cpu().double().numpy() - want)
        assert (off <= tol).all(), (off - tol).max()
    near(g.lse, lse, sum_off + 3 * e * np.abs(lse))
    near(g.entropy, entropy, sum_off * (2 + entropy) * 2 + 3 * e * size[:, 0])
    given, best = np.take_along_axis(lp, tokens.cpu().numpy(), 1), np.take_along_axis(lp, index, 1)
    near(g.logprob, given, sum_off + 3 * e * (size + np.abs(given)))
    near(g.top_logprob, best, sum_off + 3 * e * (size + np.abs(best)))
    assert np.array_equal(g.top_index.cpu().numpy(), index)
    return g


def live_tokens(V, kind, rng):
    """Which tokens stay: behind the first loads of a row, but for one wave's share, the last few, the first few, every 97th, none."""
    at = np.arange(V)
    return {"behind": at >= min(V - 3, 9000), "wave": (at // 64) % 4 != 1, "wave4": (at // 256) % 4 != 1, "wave8": (at // 512) % 4 != 2, "last": at >= V - 5, "first": at < 5,
            "some": at % 97 == 3, "none": at < 0}[kind]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["behind", "wave", "wave4", "wave8", "last", "first", "some", "none"])
@pytest.mark.parametrize("R,V", [(3, 131072), (1, 131072), (700, 2048), (2, 40003), (701, 4099), (1, 70)])
def test_token_scores_tokens_switched_off_with_the_lowest_number(R, V, kind, dtype):
    """finfo.min in place of -inf: an ordinary row over the tokens that stay, whoever of lanes, waves and parts holds nothing else."""
    rng = np.random.default_rng(V + R)
    live = live_tokens(V, kind, rng)
    x = torch.full((R, V), torch.finfo(dtype).min, dtype=dtype, device=DEV)
    x[:, torch.as_tensor(live, device=DEV)] = torch.as_tensor(rng.standard_normal((R, int(live.sum()))).astype(np.float32) * 3).to(dtype).to(DEV)
    tokens = torch.as_tensor(rng.integers(0, V, (R, 2)).astype(np.int32)).to(DEV)
    check_switched_off(x, live, tokens, min(5, V))


@pytest.mark.parametrize("V", [16384, 131072, 40003])
def test_token_scores_rising_steps_of_large_numbers(V):
    """Rows that climb from the lowest number over large steps to an ordinary end, and past it to the largest number: every step leaves the former sums nothing."""
    x = torch.empty(2, V, device=DEV)
    steps = -torch.logspace(38.5, 3, V, dtype=torch.float64)
    x[0] = steps.clamp(min=torch.finfo(F32).min).float().to(DEV)
    x[0, -100:] = torch.linspace(0, 5, 100, device=DEV)
    x[1] = x[0]
    x[1, V // 2] = torch.finfo(F32).max                                # one token has all the probability
    g = ops.token_scores(x, torch.tensor([[V - 1], [V // 2]], dtype=I32, device=DEV), 2)
    z = np.linspace(0, 5, 100).astype(np.float32).astype(np.float64)
    lse = np.log(np.exp(z).sum())
    entropy = lse - (np.exp(z - lse) * z).sum()
    e = 2.0 ** -24
    tol = (2 * 17 + 4 + V / 64 + 64) * e
    assert abs(float(g.lse[0]) - lse) <= tol + 3 * e * 15 and abs(float(g.entropy[0]) - entropy) <= tol * (2 + entropy) * 2 + 3 * e * 15
    assert abs(float(g.logprob[0, 0]) - (5 - lse)) <= tol + 3 * e * 15 and g.top_index[:, 0].tolist() == [V - 1, V // 2]
    assert float(g.lse[1]) == torch.finfo(F32).max and float(g.entropy[1]) == 0 and float(g.logprob[1, 0]) == 0


# ---- derivatives ---------------------------------------------------------------------------------------------------------------
def test_forward_mode_tangents_are_refused_on_the_gpu():
    """The compiled calls hand dual tensors back, and the Python ones refuse them; their primal values are ordinary tensors."""
    from torch.autograd.forward_ad import dual_level, make_dual, unpack_dual
    x, w, s = torch.randn(3, 32, device=DEV), torch.ones(5, 32, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV)
    plain = ops.linear_i8(x, w, s)
    with dual_level():
        d, ds = make_dual(x, torch.ones_like(x)), make_dual(s, torch.ones_like(s))
        for f, args in ((ops.linear_i8, (d, w, s)), (ops.linear_i8, (x, w, ds)), (ops.linear_i8, (x, w, s, ds)), (ops.quantize_rows_i8, (d,)), (ops.token_scores, (d,)),
                        (ops.token_scores, (d[:, 1:], None, 2))):
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                f(*args)
        assert ops._call.linear_i8(d, w, s, None) is None and ops._call.quantize_rows_i8(d) is None and ops._call.linear_i8(x, w, s, None) is not None
        assert torch.equal(ops.linear_i8(unpack_dual(d).primal, w, s), plain)
        with torch.inference_mode():                                   # forward mode is off
            assert torch.equal(ops.linear_i8(d, w, s), plain)


def test_lazily_negated_tensors_are_refused_on_the_gpu():
    x, c = torch.randn(3, 32, device=DEV), torch.zeros(2, 9, 2, 16, device=DEV)
    k, n = torch.randn(2, 3, 2, 16, device=DEV), torch.ones(2, dtype=I32, device=DEV)
    path = torch.zeros(2, 3, dtype=I32, device=DEV)
    for f, args in ((ops.quantize_rows_i8, (torch._neg_view(x),)), (ops.token_scores, (torch._neg_view(x),)), (ops.tree_commit, (k, k, torch._neg_view(c), c, path, n, n)),
                    (ops.tree_plan, (torch._neg_view(path),))):
        with pytest.raises(ValueError, match="negated"):
            f(*args)
    assert (c == 0).all()
    q, s = ops.quantize_rows_i8(torch._neg_view(x).resolve_neg())
    want = ops.quantize_rows_i8(x)
    assert torch.equal(q, -want[0]) and torch.equal(s, want[1])


# ---- caches that autograd holds ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("compiled", [True, False])
def test_tree_commit_counts_as_a_write_of_the_caches(compiled, monkeypatch):
    """A cache that a backward pass still needs cannot be written under it without a word: commits raise the tensors' version like torch's own in-place operations."""
    if not compiled:
        monkeypatch.setattr(ops, "_call", type("None_", (), {"__getattr__": lambda self, name: lambda *args: None})())
    k, path, n = torch.randn(2, 3, 2, 16, device=DEV), torch.zeros(2, 3, dtype=I32, device=DEV), torch.ones(2, dtype=I32, device=DEV)
    kc, vc = torch.zeros(2, 9, 2, 16, device=DEV), torch.zeros(2, 9, 2, 16, device=DEV)
    q = torch.ones(16, device=DEV, requires_grad=True)
    s = (kc * q).sum() + (vc[1] * q).sum()
    before = kc._version, vc._version, k._version
    ops.tree_commit(k, k, kc, vc, path, n, n)
    assert (kc._version, vc._version, k._version) == (before[0] + 1, before[1] + 1, before[2])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        s.backward()
    ops.tree_commit(k[None], k[None], kc[None], vc[None], path, n, n)
    assert kc._version == before[0] + 2
    with torch.inference_mode():                                       # tensors without a version, in and out of the mode
        kc, vc = torch.zeros(2, 9, 2, 16, device=DEV), torch.zeros(2, 9, 2, 16, device=DEV)
        ops.tree_commit(k, k, kc, vc, path, n, n)
    ops.tree_commit(k, k, kc, vc, path, n, n * 0)
    assert torch.equal(kc[:, 1], k[:, 0]) and torch.equal(kc, vc)


# ---- 8-bit integers: scales of very different sizes ----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", [(1, 1280, 40), (20, 1280, 130), (25, 77, 65), (40, 1280, 129), (64, 5120, 256), (300, 1280, 140)])
def test_linear_i8_scales_of_very_different_sizes(M, K, N, dtype):
    """Outputs of ordinary size from rows of tiny numbers and a large weight scale, or the other way round: no intermediate product leaves f32's range."""
    rng = np.random.default_rng(M + N)
    w = torch.as_tensor(rng.integers(60, 128, (N, K)).astype(np.int8)).to(DEV)
    x = torch.as_tensor((rng.random((M, K)) + 0.5).astype(np.float32)).to(DEV)
    for x_size, w_size in ((2.0 ** -115, 2.0 ** 112), (2.0 ** 115, 2.0 ** -118), (2.0 ** -60, 2.0 ** 60)):
        ws = torch.as_tensor((rng.random(N) + 0.5).astype(np.float32)).to(DEV) * w_size
        y = check_linear((x * x_size).to(dtype), w, ws, None, dtype)
        assert torch.isfinite(y).all() and (y > 1).all()


# ---- errors of others ----------------------------------------------------------------------------------------------------------
def test_an_earlier_error_of_another_call_is_not_this_calls():
    """A HIP call of the same thread that failed before (asking for a device that is not there) does not make a launch fail that succeeds."""
    parents, words, depth = torch.full((1, 3), -1, dtype=I32, device=DEV), torch.zeros(1, 3, 1, dtype=torch.int64, device=DEV), torch.full((1, 3), 7, dtype=I32, device=DEV)
    torch.cuda.synchronize()
    assert v.hip.hipSetDevice(1000) != 0 and v.hip.hipPeekAtLastError() != 0
    try:
        assert v.hip.vox_hip_tree_plan(parents.data_ptr(), None, 1, 3, words.data_ptr(), depth.data_ptr(), 0, torch.cuda.current_stream().cuda_stream) == 0, v.hip.vox_hip_last_error()
    finally:
        v.hip.hipGetLastError()
    assert depth.tolist() == [[0, 0, 0]]


# ---- f32 products in parts -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [4, 64, 128, 256])
@pytest.mark.parametrize("T,G", [(2, 4), (40, 4), (40, 1), (70, 2)])
def test_tree_attention_f32_numbers_whose_parts_are_all_as_large_as_can_be(T, G, D):
    """Many f32 rows are multiplied as three bf16 parts per number, cut off and not rounded, and three of nine products are left out: at most 2^-21 of a
    product.  Rows that see one key show it: the log-sum is the score, one product of two such numbers, and the output is the value."""
    worst = 1 + 2.0 ** -7 - 2.0 ** -23
    rng = np.random.default_rng(T + D)
    sign = lambda *s: torch.as_tensor(rng.choice([-1.0, 1.0], s)).to(F32).to(DEV)  # noqa: E731
    q = torch.zeros(1, T, G, D, device=DEV)
    q[..., 1] = worst * 4
    k, v_ = sign(1, T, 1, D) * worst, sign(1, T, 1, D) * worst * 2.0 ** torch.arange(-D // 2, D - D // 2, device=DEV).clamp(-60, 60)
    alone, depth = ops.tree_plan(torch.full((1, T), -1, dtype=I32, device=DEV))
    empty = torch.full((1, 8, 1, D), math.nan, device=DEV)
    out, lse = ops.tree_attention(q, k, v_, empty, empty, torch.zeros(1, dtype=I32, device=DEV), alone, depth, scale=0.75, return_lse=True)
    # the weight is e^(score - maximum) of a maximum that was rounded, so near 1 and not 1; (weight value) / weight: 2^-21 left out, the six products' sum
    # 6 e, the quotient e
    assert bool(((out.double() / v_.double() - 1).abs() <= 2.0 ** -21 + 7 * 2.0 ** -24).all())
    want = (q[..., 1].double() * k[..., 1].double() * 0.75).cpu().numpy()
    # left out: 2^-21; the six products' sum: 6 e; the scale and its way to base 2 and back (two constants, three products): 5 e
    assert (np.abs(lse.cpu().double().numpy() / want - 1) <= 2.0 ** -21 + 11 * 2.0 ** -24).all()


# ---- numbers of other kinds ----------------------------------------------------------------------------------------------------
def test_whole_numbers_of_other_kinds_are_taken():
    """numpy's integers and tensors of one whole number count as `top` and `window`; fractions are refused, not cut."""
    rng = np.random.default_rng(5)
    c = attn_case(5, F32, 1, 3, 4, 2, 64, 40, [33])
    x = torch.as_tensor(rng.standard_normal((3, 50)).astype(np.float32)).to(DEV)
    want, scores = ops.tree_attention(**c, window=9, scale=0.5), ops.token_scores(x, None, 3)
    for whole in (np.int64, np.int32, torch.tensor):
        assert torch.equal(ops.tree_attention(**c, window=whole(9), scale=np.float32(0.5)), want)
        assert torch.equal(ops.token_scores(x, None, whole(3)).top_index, scores.top_index)
    assert ops.token_scores(x, None, True).top_index.shape == (3, 1)
    for wrong in (9.5, "9", None):
        with pytest.raises(ValueError, match="window"):
            ops.tree_attention(**c, window=wrong)
        with pytest.raises(ValueError, match="top"):
            ops.token_scores(x, None, wrong)
    with pytest.raises(ValueError, match="scale"):
        ops.tree_attention(**c, scale="1")
