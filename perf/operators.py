"""The operators of the draft-verification step: what is timed, on which sizes, and their plain forms.

A verification pass decides in one go over several drafted tokens: the rows of all draft nodes go through the (8-bit) matrix
products, attend to the cache and to their own ancestors in the draft tree, the vocabulary rows are scored, and the accepted
path's keys and values join the cache.  Four operators, each with its cases:

  attention  attention of the nodes of a draft tree over a ring cache and over the nodes' own ancestors
  accept     ancestor sets of the tree, the accepted path, and its keys and values filed into the ring cache of every layer
  scores     log probabilities of given tokens with entropy, log-sum and the top alternatives, from rows of logits
  linear_i8  product in 8-bit integers, one scale for each row of activations and each output channel
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one stream, the real input and one drafted token behind it, a short context, the decoder's own f32 ring: the smallest pass
        dict(name="attention f32 pair", op="attention", dtype="float32", batch=1, nodes=2, heads=32, kv_heads=8, dim=128, cap=9216, length=232, window=8192),
        # a few long streams served together with a small tree each, nothing windowed: a read of the whole cache
        dict(name="attention bf16 long", op="attention", dtype="bfloat16", batch=4, nodes=24, heads=32, kv_heads=8, dim=128, cap=40960, length=40000, window=0),
        # heads of 64 without sharing, a window of 750 in a ring that has wrapped, odd counts
        dict(name="attention f16 ring", op="attention", dtype="float16", batch=3, nodes=7, heads=32, kv_heads=32, dim=64, cap=832, length=2000, window=750),
        # wide trees in f32 over a full window of the decoder's ring, wrapped several times: bound by the products
        dict(name="attention f32 wide", op="attention", dtype="float32", batch=2, nodes=64, heads=32, kv_heads=8, dim=128, cap=9216, length=30000, window=8192),
        # end of the smallest pass: two nodes, all decoder layers
        dict(name="accept f32 pair", op="accept", dtype="float32", batch=1, nodes=2, layers=26, kv_heads=8, dim=128, cap=2048, length=232),
        # end of a batched pass with trees of 63 nodes
        dict(name="accept bf16 batch", op="accept", dtype="bfloat16", batch=8, nodes=63, layers=26, kv_heads=8, dim=128, cap=1024, length=1500),
        # one decoder step's row of logits: alternatives and confidence of the token that was just chosen
        dict(name="scores f32 one row", op="scores", dtype="float32", rows=1, vocab=131072, given=1, top=8),
        # teacher-forced scoring of a 30 s clip: 386 steps
        dict(name="scores f32 clip", op="scores", dtype="float32", rows=386, vocab=131072, given=1, top=4),
        # many rows with several candidate tokens each and a long list of alternatives
        dict(name="scores bf16 many", op="scores", dtype="bfloat16", rows=1501, vocab=131072, given=8, top=32),
        # one row through the encoder's q;k;v matrix: a read of the weights
        dict(name="linear_i8 f32 row", op="linear_i8", dtype="float32", rows=1, inputs=1280, outputs=6144, bias=True),
        # a streaming chunk of 25 rows through the second matrix of the feed-forward block: few outputs, a long sum
        dict(name="linear_i8 bf16 chunk", op="linear_i8", dtype="bfloat16", rows=25, inputs=5120, outputs=1280, bias=True),
        # a long clip through the gate and up matrices: bound by the products
        dict(name="linear_i8 bf16 clip", op="linear_i8", dtype="bfloat16", rows=4099, inputs=1280, outputs=10240, bias=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "accept", "scores", "linear_i8"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "attention":
        dim = rng.choice([64, 96, 128])
        kv_heads = rng.choice([2, 4, 8])
        length = _log(rng, 1, 40000)
        window = rng.choice([0, _log(rng, 16, 8192)])
        cap = rng.choice([length + rng.randrange(0, 200), max(window, 64) + rng.randrange(0, 1024)]) if window else length + rng.randrange(0, 1024)
        batch = min(_log(rng, 1, 16), max(1, 100000 // min(length + 1, cap)))
        return dict(op=op, dtype=dtype, batch=batch, nodes=_log(rng, 1, 64), heads=kv_heads * rng.choice([1, 3, 4, 8]), kv_heads=kv_heads, dim=dim, cap=cap, length=length,
                    window=window)
    if op == "accept":
        return dict(op=op, dtype=dtype, batch=_log(rng, 1, 16), nodes=_log(rng, 1, 200), layers=rng.randrange(1, 27), kv_heads=rng.choice([2, 8]), dim=rng.choice([64, 128]),
                    cap=rng.randrange(256, 1024), length=_log(rng, 1, 3000))
    if op == "scores":
        vocab = rng.choice([rng.randrange(1000, 131073), 131072])
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, 700), vocab=vocab, given=rng.randrange(1, 9), top=rng.randrange(1, 33))
    inputs, outputs = 16 * rng.randrange(8, 321), rng.randrange(100, 10241)
    return dict(op=op, dtype=dtype, rows=min(_log(rng, 1, 4099), 50_000_000_000 // (inputs * outputs)), inputs=inputs, outputs=outputs, bias=rng.choice([True, False]))


# --------------------------------------------------------------------------------------------------------------- inputs
def _tree(g, batch, nodes):
    """Random draft trees: a node's parent is the cache's end (-1) or an earlier node, mostly a near one.  All but the first tree may be shorter."""
    at = torch.arange(nodes, device=DEV)
    back = (torch.rand(batch, nodes, device=DEV, generator=g).square() * 4).long() + 1
    parents = (at - back).clamp(min=-1)
    n = nodes - (torch.rand(batch, device=DEV, generator=g) * max(1, nodes // 3)).long()
    n[0] = nodes
    return parents.int(), n.int()


def _ancestors(parents, n_nodes):
    """[batch, nodes, nodes] truth values (node j is i or an ancestor of i) and the depths; nothing and -1 for nodes that are not there."""
    batch, nodes = parents.shape
    at = torch.arange(nodes, device=parents.device)
    here = at < n_nodes[:, None]
    reach = ((parents[:, :, None] == at) | (at[:, None] == at)).float()
    for _ in range(max(1, (nodes - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    anc = (reach > 0) & here[:, :, None]
    depth = torch.where(here, anc.sum(-1) - 1, -1)
    return anc, depth.int()


def _words(anc):
    """Truth values to 64-bit words, bit j % 64 of word j // 64."""
    batch, nodes, _ = anc.shape
    words = (nodes + 63) // 64
    bits = torch.zeros(batch, nodes, words * 64, dtype=torch.int64, device=anc.device)
    bits[:, :, :nodes] = anc
    return (bits.view(batch, nodes, words, 64) << torch.arange(64, device=anc.device)).sum(-1)


def _lengths(g, batch, length):
    n = (length * (1 - 0.4 * torch.rand(batch, device=DEV, generator=g))).int().clamp(min=1)
    n[0] = length
    return n


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, device=DEV, generator=g, dtype=torch.float32 if dtype == torch.float32 else dtype) * scale).to(dtype)

    s = dict(case=case)
    if case["op"] == "attention":
        B, T, H, Hk, D = (case[k] for k in ("batch", "nodes", "heads", "kv_heads", "dim"))
        s["q"], s["k"], s["v"] = randn(B, T, H, D, scale=1.5), randn(B, T, Hk, D), randn(B, T, Hk, D)
        s["k_cache"], s["v_cache"] = randn(B, case["cap"], Hk, D), randn(B, case["cap"], Hk, D)
        s["cache_len"] = _lengths(g, B, case["length"])
        anc, s["depth"] = _ancestors(*_tree(g, B, T))
        s["ancestors"] = _words(anc)
    elif case["op"] == "accept":
        L, B, T, Hk, D = (case[k] for k in ("layers", "batch", "nodes", "kv_heads", "dim"))
        s["parents"], s["n_nodes"] = _tree(g, B, T)
        s["k"], s["v"] = randn(L, B, T, Hk, D), randn(L, B, T, Hk, D)
        s["k_cache"], s["v_cache"] = randn(L, B, case["cap"], Hk, D), randn(L, B, case["cap"], Hk, D)
        s["cache_len"] = _lengths(g, B, case["length"])
        # drafts over a small set of tokens, most of which the model agrees with, so that paths of several nodes are accepted
        s["tokens"] = torch.randint(1000, 1003, (B, T), device=DEV, generator=g, dtype=torch.int32)
        s["choices"] = torch.randint(1000, 1003, (B, T), device=DEV, generator=g, dtype=torch.int32)
        s["root_choice"] = s["tokens"][:, 0].clone()
    elif case["op"] == "scores":
        R, V = case["rows"], case["vocab"]
        s["logits"] = randn(R, V, scale=2.5)
        s["logits"][:, V // 2: V // 2 + 7] = -math.inf  # tokens that are switched off
        peak = torch.randint(0, V, (R, 1), device=DEV, generator=g)
        s["logits"].scatter_(1, peak, (torch.rand(R, 1, device=DEV, generator=g) * 20 + 5).to(dtype))  # confident rows and others
        s["tokens"] = torch.cat([peak, torch.randint(0, V, (R, case["given"] - 1), device=DEV, generator=g)], 1).int()
    else:
        M, K, N = case["rows"], case["inputs"], case["outputs"]
        s["x"] = randn(M, K)
        s["x"][:, :: 97] *= 8  # a few loud channels, as activations have them
        s["w"] = torch.randint(-127, 128, (N, K), device=DEV, generator=g, dtype=torch.int8)
        s["w_scale"] = (torch.rand(N, device=DEV, generator=g) + 0.5) / (127 * math.sqrt(K))
        s["bias"] = randn(N) if case["bias"] else None
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _positions(length, cap, window):
    """[batch, most] positions that any node may see, their ring slots, and which are there at all."""
    low = (length - cap).clamp(min=0)
    if window > 0:
        low = torch.maximum(low, length - window + 1)
    most = int((length - low).max())
    pos = low[:, None] + torch.arange(most, device=length.device)
    return pos, pos % cap, pos < length[:, None]


def _attention(s):
    c = s["case"]
    B, T, H, Hk, D = (c[k] for k in ("batch", "nodes", "heads", "kv_heads", "dim"))
    G, window = H // Hk, c["window"]
    length, depth = s["cache_len"].long(), s["depth"].long()
    pos, slot, there = _positions(length, c["cap"], window)
    row = torch.arange(B, device=DEV)[:, None]
    k = torch.cat([s["k_cache"][row, slot], s["k"]], 1).float().permute(0, 2, 3, 1).contiguous()
    v = torch.cat([s["v_cache"][row, slot], s["v"]], 1).float().transpose(1, 2).contiguous()
    at = torch.arange(T, device=DEV)
    seen = (s["ancestors"][:, :, at // 64] >> (at % 64)) & 1 > 0
    cached = there[:, None, :] & (depth >= 0)[:, :, None]
    if window > 0:
        cached = cached & (pos[:, None, :] > (length[:, None] + depth)[:, :, None] - window)
        seen = seen & (depth[:, None, :] > depth[:, :, None] - window)
    mask = torch.cat([cached, seen], 2)[:, None, :, None, :]
    q = s["q"].float().view(B, T, Hk, G, D).transpose(1, 2).reshape(B, Hk, T * G, D)
    x = (torch.matmul(q, k) / math.sqrt(D)).view(B, Hk, T, G, -1).masked_fill(~mask, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m.masked_fill(m == -math.inf, 0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul((p / total.masked_fill(total == 0, 1)).view(B, Hk, T * G, -1), v)
    o = o.view(B, Hk, T, G, D).transpose(1, 2).reshape(B, T, H, D).to(s["q"].dtype)
    lse = (m + torch.log(total)).squeeze(-1).transpose(1, 2).reshape(B, T, H)
    return o, lse


def _accept(s):
    c = s["case"]
    B, T = c["batch"], c["nodes"]
    parents, n_nodes = s["parents"].long(), s["n_nodes"].long()
    anc, depth = _ancestors(parents, n_nodes)
    want = torch.where(parents < 0, s["root_choice"][:, None], torch.gather(s["choices"], 1, parents.clamp(min=0)))
    match = (s["tokens"] == want) & (depth >= 0)
    at = torch.arange(T, device=DEV)
    earlier = (parents[:, :, None] == parents[:, None, :]) & (at[None, :] < at[:, None]) & match[:, None, :]
    match = match & ~earlier.any(-1)  # of equal drafts behind the same node the lowest counts
    kept = (~anc | match[:, None, :]).all(-1) & (depth >= 0)
    count = kept.sum(1)
    path = torch.full((B, T + 1), -1, dtype=torch.int64, device=DEV)
    path.scatter_(1, torch.where(kept, depth.long(), T), at.expand(B, T))  # column T takes the nodes that are not kept
    path = path[:, :T].contiguous()
    last = torch.gather(path, 1, (count - 1).clamp(min=0)[:, None])
    after = torch.where(count > 0, torch.gather(s["choices"], 1, last.clamp(min=0)).squeeze(1), s["root_choice"])
    length = s["cache_len"].long()
    b, j = torch.nonzero(path >= 0, as_tuple=True)
    node, slot = path[b, j], (length[b] + j) % c["cap"]
    s["k_cache"][:, b, slot] = s["k"][:, b, node]
    s["v_cache"][:, b, slot] = s["v"][:, b, node]
    return _words(anc), depth, path.int(), count.int(), after.int(), (length + count).int(), s["k_cache"], s["v_cache"]


def _scores(s):
    c = s["case"]
    x = s["logits"].double()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    logprob = torch.gather(x, 1, s["tokens"].long()) - lse
    entropy = lse.squeeze(1) - (torch.where(e > 0, x, 0) * e).sum(1) / total.squeeze(1)
    value, index = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    return logprob.float(), entropy.float(), lse.squeeze(1).float(), index[:, : c["top"]].int(), (value[:, : c["top"]].double() - lse).float()


def _linear_i8(s):
    x = s["x"].double()
    scale = (x.abs().amax(1, keepdim=True).float() / 127).clamp(min=2.0 ** -126)
    q = torch.round(x / scale.double())
    y = torch.matmul(q, s["w"].double().t()) * scale.double() * s["w_scale"].double()
    return (y if s["bias"] is None else y + s["bias"].double()).to(s["x"].dtype)


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"attention": _attention, "accept": _accept, "scores": _scores, "linear_i8": _linear_i8}[op](s)
    from voxtral_c_amd import ops

    if op == "attention":
        return ops.tree_attention(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["cache_len"], s["ancestors"], s["depth"], window=s["case"]["window"], return_lse=True)
    if op == "accept":
        ancestors, depth = ops.tree_plan(s["parents"], s["n_nodes"])
        path, count, after, length = ops.tree_accept(s["tokens"], s["choices"], s["root_choice"], s["parents"], ancestors, depth, s["cache_len"])
        ops.tree_commit(s["k"], s["v"], s["k_cache"], s["v_cache"], path, count, s["cache_len"])
        return ancestors, depth, path, count, after, length, s["k_cache"], s["v_cache"]
    if op == "scores":
        r = ops.token_scores(s["logits"], s["tokens"], top=s["case"]["top"])
        return r.logprob, r.entropy, r.lse, r.top_index, r.top_logprob
    return ops.linear_i8(s["x"], s["w"], s["w_scale"], s["bias"])


# ----------------------------------------------------------------------------------------------------- work and exactness
def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "attention":
        B, T, H, Hk, D = (case[k] for k in ("batch", "nodes", "heads", "kv_heads", "dim"))
        # lengths are between 0.6 and 1 of the stated one, trees between 2/3 and 1: 0.8 and 0.83 on average behind the first
        share = lambda mean: (1 + mean * (B - 1)) / B  # noqa: E731
        keys = min(case["length"] * share(0.8), case["cap"], case["window"] or 1 << 40)
        nodes = T * share(0.83)
        return {"bytes": B * size * (2 * T * H * D + 2 * (keys + T) * Hk * D) + B * T * (H * 4 + 8 * ((T + 63) // 64) + 4), "flops": 4 * B * nodes * H * D * (keys + min(8, nodes))}
    if case["op"] == "accept":
        B, T = case["batch"], case["nodes"]
        rows = 2 * case["layers"] * case["kv_heads"] * case["dim"] * size
        return {"bytes": B * (min(T, 3) * rows * 2 + T * (8 * ((T + 63) // 64) + 20)), "flops": B * T * 8}
    if case["op"] == "scores":
        return {"bytes": case["rows"] * (case["vocab"] * size + 8 * (case["given"] + case["top"] + 1)), "flops": case["rows"] * case["vocab"] * 6}
    M, K, N = case["rows"], case["inputs"], case["outputs"]
    return {"bytes": M * K * size + N * K + 4 * N + M * N * size, "flops": 2 * M * K * N}


def _exact_attention(s):
    """Sequence by sequence and head by head in 64 bits, over the keys that a sequence holds."""
    c, out, lse = s["case"], [], []
    G, window, at = c["heads"] // c["kv_heads"], c["window"], torch.arange(c["nodes"], device=DEV)
    for b in range(c["batch"]):
        n, d = int(s["cache_len"][b]), s["depth"][b].double()
        first = max(0, n - c["cap"], n - window + 1 if window > 0 else 0)
        p = torch.arange(first, n, device=DEV)
        reach = (n + d[:, None] - p) < window if window > 0 else torch.ones(len(at), len(p), dtype=torch.bool, device=DEV)
        bits = torch.stack([(s["ancestors"][b, :, j // 64] >> (j % 64)) & 1 for j in range(c["nodes"])], 1) == 1
        near = d[:, None] - d[None, :] < window if window > 0 else torch.ones_like(bits)
        allowed = torch.cat([reach & (d >= 0)[:, None], bits & near], 1)
        rows, sums = [], []
        for h in range(c["heads"]):
            kk = torch.cat([s["k_cache"][b, p % c["cap"], h // G], s["k"][b, :, h // G]]).double()
            vv = torch.cat([s["v_cache"][b, p % c["cap"], h // G], s["v"][b, :, h // G]]).double()
            x = (s["q"][b, :, h].double() @ kk.t().contiguous()) * c["dim"] ** -0.5
            x = torch.where(allowed, x, torch.full_like(x, -math.inf))
            t = torch.logsumexp(x, 1)
            w = torch.where(allowed.any(1)[:, None], torch.exp(x - t[:, None]), torch.zeros_like(x))
            rows.append(w @ vv)
            sums.append(t)
        out.append(torch.stack(rows, 1))
        lse.append(torch.stack(sums, 1))
    return torch.stack(out), torch.stack(lse)


def _exact_accept(s):
    """The walk down the tree, node by node, on the host; rows of numbers are copied, so they are their own 64-bit value."""
    c = s["case"]
    parents, n_nodes, tokens, choices, root, length = (s[k].cpu().tolist() for k in ("parents", "n_nodes", "tokens", "choices", "root_choice", "cache_len"))
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    for b in range(c["batch"]):
        node, want, j = -1, root[b], 0
        while True:
            node = next((i for i in range(n_nodes[b]) if parents[b][i] == node and tokens[b][i] == want), None)
            if node is None:
                break
            slot = (length[b] + j) % c["cap"]
            kc[:, b, slot], vc[:, b, slot] = s["k"][:, b, node].double(), s["v"][:, b, node].double()
            want, j = choices[b][node], j + 1
    return None, None, None, None, None, None, kc, vc


def _exact_scores(s):
    x = s["logits"].double()
    p = torch.softmax(x, 1)
    lp = torch.log_softmax(x, 1)
    entropy = -(torch.where(p > 0, lp, torch.zeros_like(lp)) * p).sum(1)
    top = lp.topk(s["case"]["top"], 1).values
    return lp.gather(1, s["tokens"].long()), entropy, torch.logsumexp(x, 1), None, top


def _exact_linear_i8(s):
    """Rows in turn; the scale is the number that 32 bits hold, as the definition has it."""
    step, rows = 512, []
    w = (s["w"].double() * s["w_scale"].double()[:, None]).t().contiguous()
    for i in range(0, s["case"]["rows"], step):
        x = s["x"][i: i + step].double()
        scale = torch.maximum((x.abs().max(1).values.float() / 127.0).double(), torch.tensor(2.0 ** -126, dtype=torch.float64, device=DEV))
        t = x / scale[:, None]
        low = torch.floor(t)
        up = (t - low > 0.5) | ((t - low == 0.5) & (low % 2 == 1))
        rows.append(((low + up) * scale[:, None]) @ w)
    y = torch.cat(rows)
    return y if s["bias"] is None else y + s["bias"].double()


def exact(case, seed):
    return {"attention": _exact_attention, "accept": _exact_accept, "scores": _exact_scores, "linear_i8": _exact_linear_i8}[case["op"]](prepare(case, seed))
