"""Plain 64-bit forms of the draft-verification operators (vox_hip_ops.h), written loop by loop from their definitions, on the CPU."""
import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step of a rounding, relative


def random_tree(rng, B, T, shorter=True):
    parents = np.stack([[rng.integers(-1, i) if rng.random() < 0.5 else i - 1 - min(i, int(rng.integers(0, 3))) for i in range(T)] for _ in range(B)]).astype(np.int32)
    n = np.array([T if b == 0 or not shorter else rng.integers(0, T + 1) for b in range(B)], np.int32)
    return parents, n


def plan(parents, n_nodes):
    """(list of ancestor sets, depths): None / -1 for nodes that are not there."""
    B, T = parents.shape
    sets, depth = [], np.full((B, T), -1, np.int32)
    for b in range(B):
        s = []
        for i in range(T):
            p = int(parents[b, i])
            ok = i < n_nodes[b] and -1 <= p < i and (p < 0 or s[p] is not None)
            s.append(({i} | (s[p] if p >= 0 else set())) if ok else None)
            if ok:
                depth[b, i] = len(s[i]) - 1
        sets.append(s)
    return sets, depth


def words(sets, T):
    B, W = len(sets), (T + 63) // 64
    out = np.zeros((B, T, W), np.uint64)
    for b in range(B):
        for i in range(T):
            for j in sets[b][i] or ():
                out[b, i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def attention(q, k, v, kc, vc, cache_len, mask_words, depth, scale, window):
    """(out, lse, err, lse_err, mean): 64-bit values, how far f32 arithmetic may be off per row, and the weighted mean of |v| per element."""
    q, k, v, kc, vc = (t.detach().cpu().double().numpy() for t in (q, k, v, kc, vc))
    B, T, H, D = q.shape
    Hk, cap = k.shape[2], kc.shape[1]
    out, lse = np.zeros((B, T, H, D)), np.full((B, T, H), -np.inf)
    err, lerr, mean = np.zeros((B, T, H, 1)), np.zeros((B, T, H)), np.zeros((B, T, H, D))
    e = 2.0 ** -24
    for b in range(B):
        n = max(int(cache_len[b]), 0)
        for i in range(T):
            d = int(depth[b, i])
            cached = [p for p in range(max(0, n - cap), n) if d >= 0 and (window <= 0 or p > n + d - window)]
            nodes = [j for j in range(T) if d >= 0 and (int(mask_words[b, i, j // 64]) >> (j % 64)) & 1 and (window <= 0 or depth[b, j] > d - window)]
            rows = [p % cap for p in cached]
            if not rows and not nodes:
                continue
            for h in range(H):
                g = h // (H // Hk)
                K, V = np.concatenate([kc[b, rows, g], k[b, nodes, g]]), np.concatenate([vc[b, rows, g], v[b, nodes, g]])
                s = K @ q[b, i, h] * scale
                m = s.max()
                p = np.exp(s - m)
                out[b, i, h], lse[b, i, h] = p @ V / p.sum(), m + np.log(p.sum())
                mean[b, i, h] = p @ np.abs(V) / p.sum()
                # f32: a score of D products is off by (D + 4) e of the sum of their sizes; the exponential's argument by 2 e of its size on top and the
                # exponential by 4 e; sums of n terms, rescaling by the running maximum and the division by (n + 16) e.  Relative errors of the
                # weights move out by twice their largest times the largest |v|.
                ds = (D + 4) * e * (np.abs(K) @ np.abs(q[b, i, h])).max() * abs(scale) + 4 * e * (np.abs(s).max() + abs(m)) + 4 * e
                err[b, i, h] = (2 * ds + (len(s) + 16) * e) * np.abs(V).max()
                lerr[b, i, h] = ds + (len(s) + 16) * e + 2 * e * abs(lse[b, i, h])
    return out, lse, err, lerr, mean


def attention_bound(out, err, mean, dtype):
    """The arithmetic's part, the storage rounding of out, and, for the 16-bit types, one rounding of every weight in front of its product."""
    h = HALF[dtype]
    return err + 1.01 * h * np.abs(out) + (0 if dtype == torch.float32 else 1.01 * h * mean) + 1e-30


def accept(parents, n_nodes, tokens, choices, root, cache_len):
    B, T = parents.shape
    sets, _ = plan(parents, n_nodes)
    path, n, after = np.full((B, T), -1, np.int32), np.zeros(B, np.int32), np.zeros(B, np.int32)
    for b in range(B):
        node, want = -1, int(root[b])
        while True:
            nxt = [i for i in range(T) if sets[b][i] is not None and parents[b, i] == node and tokens[b, i] == want]
            if not nxt:
                break
            node = nxt[0]
            path[b, n[b]] = node
            n[b] += 1
            want = int(choices[b, node])
        after[b] = want
    return path, n, after, (np.maximum(cache_len, 0) + n).astype(np.int32)


def quantize(x):
    """(whole numbers, scales) in exact arithmetic: 64-bit quotients of two f32 numbers separate every border."""
    x = x.detach().cpu().float().numpy()
    amax = np.abs(x).max(1)
    bad = ~np.isfinite(x).all(1)
    scale = np.maximum((np.where(bad, 0, amax).astype(np.float32) / np.float32(127)), np.float32(2.0 ** -126)).astype(np.float32)
    with np.errstate(invalid="ignore"):
        q = np.rint(np.where(bad[:, None], 0, x).astype(np.float64) / scale[:, None].astype(np.float64)).astype(np.int64)
    return q, np.where(bad, np.float32(np.nan), scale)
