"""Serving operators around a decode step: their cases, inputs, plain forms and exact values.

Four operators that a serving loop chains: attention over packed prompts of
different lengths, attention of a tree of drafted tokens over a KV cache, the
commit of the accepted branch into the cache, and log probabilities of given
tokens.  ``run`` computes them in elementary torch operations (``own`` false)
or through ``torch2iron_b200.operators`` (``own`` true); ``exact`` computes
them in 64 bits from their definitions.

Head layouts are those of the benchmark configurations (16 or 32 query heads
over 8 key heads of 128, 32 over 8 of 64) and vocabularies theirs (151936 and
128256); lengths run from one token to a long prompt or context.
"""

import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HEADS = {"16x8x128": (16, 8, 128), "32x8x128": (32, 8, 128), "32x8x64": (32, 8, 64)}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a few chat turns arriving together: latency counts
        {"name": "packed_short", "op": "packed", "heads": "16x8x128", "type": "bf16", "seqs": 8, "longest": 37,
         "spread": 0.9, "prefix": 0},
        # one prefill step of a busy server: ragged prompts, no padding
        {"name": "packed_ragged", "op": "packed", "heads": "32x8x128", "type": "bf16", "seqs": 24, "longest": 1501,
         "spread": 0.97, "prefix": 0},
        # one long document beside two shorter ones
        {"name": "packed_long", "op": "packed", "heads": "32x8x128", "type": "bf16", "seqs": 3, "longest": 12001,
         "spread": 0.7, "prefix": 0},
        # suffixes of cached prompts (and single tokens) attending their cache rows
        {"name": "packed_suffix", "op": "packed", "heads": "32x8x64", "type": "fp16", "seqs": 17, "longest": 200,
         "spread": 0.995, "prefix": 3000},
        # one user, a small tree over a short context: latency counts
        {"name": "tree_one_user", "op": "tree", "heads": "16x8x128", "type": "bf16", "rows": 1, "nodes": 8,
         "context": 437},
        # a batch of ordinary trees over ordinary contexts
        {"name": "tree_batch", "op": "tree", "heads": "32x8x64", "type": "bf16", "rows": 32, "nodes": 21,
         "context": 4099},
        # a wide tree over two long documents
        {"name": "tree_long", "op": "tree", "heads": "32x8x128", "type": "bf16", "rows": 2, "nodes": 63,
         "context": 60001},
        # the accepted branch of one user's tree, all layers of the small model
        {"name": "commit_one_user", "op": "commit", "heads": "16x8x128", "type": "bf16", "layers": 28, "rows": 1,
         "nodes": 8, "context": 256},
        # the accepted branches of a batch of wide trees
        {"name": "commit_batch", "op": "commit", "heads": "32x8x64", "type": "bf16", "layers": 16, "rows": 64,
         "nodes": 48, "context": 384},
        # the log probability of one sampled token, with twenty alternatives
        {"name": "logprobs_one_row", "op": "logprobs", "type": "fp32", "rows": 1, "vocab": 151936, "top": 20,
         "masked": 0.0},
        # a decode batch under a grammar: half of the vocabulary masked
        {"name": "logprobs_masked", "op": "logprobs", "type": "bf16", "rows": 65, "vocab": 128256, "top": 5,
         "masked": 0.5},
        # scoring a chunk of a prompt
        {"name": "logprobs_score", "op": "logprobs", "type": "fp32", "rows": 1500, "vocab": 151936, "top": 1,
         "masked": 0.0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["packed", "packed", "tree", "tree", "commit", "logprobs"])
    heads = rng.choice(sorted(HEADS))
    kind = rng.choice(["bf16", "bf16", "fp16"])
    if op == "packed":
        prefix = rng.choice([0, 0, _log(rng, 1, 4000)])
        longest = _log(rng, 1, 6000)
        seqs = _log(rng, 1, max(1, min(40, 16000 // longest)))
        return {"op": op, "heads": heads, "type": kind, "seqs": seqs, "longest": longest,
                "spread": rng.uniform(0.0, 1.0), "prefix": prefix}
    if op == "tree":
        context = _log(rng, 1, 50000)
        rows = _log(rng, 1, max(1, min(64, 100000 // context)))
        return {"op": op, "heads": heads, "type": kind, "rows": rows, "nodes": _log(rng, 1, 130), "context": context}
    if op == "commit":
        return {"op": op, "heads": heads, "type": kind, "layers": rng.randint(1, 36), "rows": _log(rng, 1, 32),
                "nodes": _log(rng, 1, 130), "context": rng.randint(135, 400)}
    vocab = _log(rng, 37, 151936)
    return {"op": op, "type": rng.choice(["fp32", "bf16", "fp16"]), "rows": _log(rng, 1, 1000), "vocab": vocab,
            "top": rng.choice([0, 1, 5, 20, min(32, vocab)]), "masked": rng.choice([0.0, 0.3, 0.9])}


def _lengths(case):
    """Query lengths of the sequences: from ``longest`` down to ``(1 - spread) longest``, out of order."""
    n, longest = case["seqs"], case["longest"]
    got = [max(1, round(longest * (1.0 - case["spread"] * (i / max(1, n - 1)) ** 0.7))) for i in range(n)]
    return [got[(i * 5 + 2) % n] if n % 5 else got[(i * 3 + 1) % n] for i in range(n)]


def _prefixes(case):
    """Cached keys before each sequence's first query."""
    return [case["prefix"] * (1 + 3 * i) // (1 + 3 * (case["seqs"] - 1)) for i in range(case["seqs"])]


def _contexts(case):
    """Cached keys of each row."""
    n, c = case["rows"], case["context"]
    return [max(0, c - (c * ((i * 7) % n)) // (2 * n)) for i in range(n)]


def _nodes(case):
    """Live nodes of each row's tree."""
    return [max(1, case["nodes"] - (i * 3) % max(1, case["nodes"] // 4)) for i in range(case["rows"])]


def _accepted(case):
    """Accepted nodes of each row's tree, the root among them."""
    return [1 + (i * 5 + 3) % min(n, 8) for i, n in enumerate(_nodes(case))]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _trees(rng, rows, nodes, live, chain):
    """Random trees [rows, nodes]: node 0 is the root, parents precede their
    children; ``chain[b]`` nodes of row b form one branch from the root."""
    parents = np.full((rows, nodes), -1, np.int32)
    on_chain = []
    for b in range(rows):
        n = live[b]
        for i in range(1, n):
            parents[b, i] = rng.integers(max(0, i - 6), i)
        branch = np.concatenate([[0], 1 + np.sort(rng.choice(max(1, n - 1), chain[b] - 1, replace=False))]) \
            if chain[b] > 1 else np.array([0])
        parents[b, branch[1:]] = branch[:-1]
        on_chain.append(branch)
    return parents, on_chain


def _mask_words(parents, live):
    """Ancestor-or-self bits [rows, nodes, words] of the live nodes."""
    rows, nodes = parents.shape
    words = np.zeros((rows, nodes, (nodes + 63) // 64), np.uint64)
    for b in range(rows):
        for i in range(live[b]):
            if parents[b, i] >= 0:
                words[b, i] = words[b, parents[b, i]]
            words[b, i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
    return words.view(np.int64)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    dt = TYPES[case["type"]]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).mul_(scale).to(dt)

    def ints(values):
        return torch.tensor(np.asarray(values), dtype=torch.int32, device=dev)

    s = {"case": dict(case)}
    op = case["op"]
    if op != "logprobs":
        nh, nkv, hd = HEADS[case["heads"]]
        s.update(nh=nh, nkv=nkv, hd=hd)
    if op == "packed":
        n = _lengths(case)
        pre = _prefixes(case)
        total = sum(n)
        s.update(n=n, k_n=[a + b for a, b in zip(n, pre)], q=randn(total, nh, hd, scale=1.5),
                 q_start=ints(np.concatenate([[0], np.cumsum(n)])),
                 out=torch.zeros(total, nh, hd, device=dev, dtype=dt), lse=torch.zeros(total, nh, device=dev))
        if case["prefix"]:
            max_ctx = -(-max(s["k_n"]) // 64) * 64
            s.update(max_ctx=max_ctx, k=randn(len(n), nkv, max_ctx, hd), v=randn(len(n), nkv, max_ctx, hd),
                     k_len=ints(s["k_n"]))
        else:
            s.update(max_ctx=None, k=randn(total, nkv, hd), v=randn(total, nkv, hd))
    elif op == "tree":
        B, T = case["rows"], case["nodes"]
        live, ctx = _nodes(case), _contexts(case)
        max_ctx = -(-(max(ctx) + T) // 64) * 64
        parents, _ = _trees(rng, B, T, live, [min(3, x) for x in live])
        s.update(live=live, ctx=ctx, max_ctx=max_ctx, q=randn(B, T, nh, hd, scale=1.5),
                 k_cache=randn(B, nkv, max_ctx, hd), v_cache=randn(B, nkv, max_ctx, hd),
                 k_draft=randn(B, T, nkv, hd), v_draft=randn(B, T, nkv, hd), ctx_len=ints(ctx), num_nodes=ints(live),
                 mask=torch.tensor(_mask_words(parents, live), device=dev),
                 out=torch.zeros(B, T, nh, hd, device=dev, dtype=dt), lse=torch.zeros(B, T, nh, device=dev))
    elif op == "commit":
        L, B, T = case["layers"], case["rows"], case["nodes"]
        live, take, max_ctx = _nodes(case), _accepted(case), -(-case["context"] // 64) * 64
        parents, branch = _trees(rng, B, T, live, take)
        tokens = rng.integers(1000, 120000, (B, T)).astype(np.int32)
        predicted = rng.integers(200000, 300000, (B, T)).astype(np.int32)   # agrees with no draft
        for b, nodes in enumerate(branch):
            tokens[b, nodes] = rng.integers(0, 1000, len(nodes))
            predicted[b, nodes[:-1]] = tokens[b, nodes[1:]]
        s.update(tokens=ints(tokens), parents=ints(parents), predicted=ints(predicted), num_nodes=ints(live),
                 ctx_len=ints([max(0, case["context"] - T - 3 * i % 64) for i in range(B)]),
                 k_drafts=randn(L, B, T, nkv, hd), v_drafts=randn(L, B, T, nkv, hd),
                 k_caches=randn(L, B, nkv, max_ctx, hd), v_caches=randn(L, B, nkv, max_ctx, hd), max_ctx=max_ctx,
                 path=torch.zeros(B, T, dtype=torch.int32, device=dev),
                 **{k: torch.zeros(B, dtype=torch.int32, device=dev) for k in ("num_accepted", "next_token", "new_len")})
    else:
        M, V, K = case["rows"], case["vocab"], case["top"]
        x = torch.randn(M, V, generator=g, device=dev).mul_(2.0)
        # a few likely tokens in each row, as a language model's logits have them
        few = min(V, 40)
        x.scatter_add_(1, torch.randint(0, V, (M, few), generator=g, device=dev),
                       torch.rand(M, few, generator=g, device=dev).mul_(12.0))
        tokens = x.topk(min(V, 30), dim=1).indices
        tokens = tokens.gather(1, torch.randint(0, min(V, 30), (M, 1), generator=g, device=dev))[:, 0]
        if case["masked"]:
            hide = torch.rand(M, V, generator=g, device=dev) < case["masked"]
            hide.scatter_(1, tokens[:, None], False)
            x.masked_fill_(hide, -math.inf)
        f32 = torch.float32
        s.update(logits=x.to(dt), tokens=tokens.to(torch.int32), logprob=torch.zeros(M, dtype=f32, device=dev),
                 entropy=torch.zeros(M, dtype=f32, device=dev),
                 top_logprob=torch.zeros(M, K, dtype=f32, device=dev) if K else None,
                 top_index=torch.zeros(M, K, dtype=torch.int32, device=dev) if K else None)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)[s["case"]["op"]](s)


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(hd)) v over the seen keys, in 32 bits.

    q [S, n, nh, hd], k and v [S, m, nkv, hd], seen [S, n, m] -> out [S, n, nh, hd], lse [S, n, nh]."""
    S, n, nh, hd = q.shape
    nkv = k.shape[2]
    q = q.float().reshape(S, n, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(S, nkv, nh // nkv * n, hd)
    x = torch.matmul(q, k.float().permute(0, 2, 3, 1)) * (1.0 / math.sqrt(hd))
    x = x.reshape(S, nkv, nh // nkv, n, -1).masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isfinite(m), m, 0.0))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(S, nkv, nh // nkv * n, -1), v.float().permute(0, 2, 1, 3))
    o = o.reshape(S, nkv, nh // nkv, n, hd) / torch.where(l > 0, l, 1.0)
    lse = torch.log(l) + torch.where(torch.isfinite(m), m, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(S, n, nh, hd), lse[..., 0].permute(0, 3, 1, 2).reshape(S, n, nh)


MOST_SCORES = 1 << 29   # scores held at once


def _packed_plain(s):
    q, n, k_n, dev = s["q"], s["n"], s["k_n"], s["q"].device
    S, nh = len(n), s["nh"]
    start = np.concatenate([[0], np.cumsum(n)])
    if S * nh * max(n) * max(k_n) <= MOST_SCORES:      # all sequences at once, padded to the longest
        i, j = torch.arange(max(n), device=dev), torch.arange(max(k_n), device=dev)
        tn = torch.tensor(n, device=dev)[:, None]
        tk = torch.tensor(k_n, device=dev)[:, None]
        first = s["q_start"][:-1, None].long()
        live = i[None] < tn
        at = torch.where(live, first + i[None], 0)
        seen = j[None, None] <= (tk - tn)[:, :, None] + i[None, :, None]
        if s["max_ctx"] is None:
            kat = torch.where(j[None] < tk, first + j[None], 0)
            k, v = s["k"][kat], s["v"][kat]
        else:
            k, v = (s[x][:, :, :max(k_n)].transpose(1, 2) for x in ("k", "v"))
        o, lse = _attend(q[at], k, v, seen & live[:, :, None])
        return {"out": o[live].to(q.dtype), "lse": lse[live]}
    out, lse = torch.empty_like(s["out"]), torch.empty_like(s["lse"])
    for b in range(S):                                 # long ones: a block of queries of one sequence at a time
        if s["max_ctx"] is None:
            k, v = (s[x][None, start[b]:start[b + 1]] for x in ("k", "v"))
        else:
            k, v = (s[x][b:b + 1, :, :k_n[b]].transpose(1, 2) for x in ("k", "v"))
        step = max(1, MOST_SCORES // (nh * k_n[b]))
        for c in range(0, n[b], step):
            e = min(c + step, n[b])
            last = k_n[b] - n[b] + e
            seen = torch.arange(last, device=dev)[None, None] <= \
                k_n[b] - n[b] + torch.arange(c, e, device=dev)[None, :, None]
            o, l = _attend(q[None, start[b] + c:start[b] + e], k[:, :last], v[:, :last], seen)
            out[start[b] + c:start[b] + e] = o[0].to(q.dtype)
            lse[start[b] + c:start[b] + e] = l[0]
    return {"out": out, "lse": lse}


def _packed_own(s):
    from torch2iron_b200.operators import PackedAttention
    op = PackedAttention(tokens=s["q"].shape[0], num_seqs=len(s["n"]), num_kv_groups=s["nkv"],
                         q_heads_per_group=s["nh"] // s["nkv"], head_dim=s["hd"], max_ctx=s["max_ctx"],
                         dtype=s["q"].dtype)
    op(s["q"], s["k"], s["v"], s["q_start"], s["out"], k_len=s.get("k_len"), lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _tree_plain(s):
    B, T, nh, hd = s["q"].shape
    dev = s["q"].device
    bits = torch.arange(T, device=dev)
    inside = (s["mask"][:, :, bits // 64] >> (bits % 64)) & 1 == 1                        # [B, T, T]
    live = torch.arange(T, device=dev)[None] < s["num_nodes"][:, None]
    c = max(s["ctx"])
    step = max(1, MOST_SCORES // (nh * T * (c + T)))
    out, lse = torch.zeros_like(s["out"]), torch.zeros_like(s["lse"])
    for b in range(0, B, step):                                                            # a few rows at a time
        r = slice(b, min(b + step, B))
        before = torch.arange(c, device=dev)[None] < s["ctx_len"][r, None]
        before = before[:, None].expand(-1, T, -1)
        k, v = (torch.cat([s[x + "_cache"][r, :, :c].transpose(1, 2), s[x + "_draft"][r]], 1) for x in ("k", "v"))
        seen = torch.cat([before, inside[r] & live[r, None]], 2)
        o, l = _attend(s["q"][r], k, v, seen)
        out[r] = torch.where(live[r, :, None, None], o.to(out.dtype), 0)
        lse[r] = torch.where(live[r, :, None], l, 0)
    return {"out": out, "lse": lse}


def _tree_own(s):
    from torch2iron_b200.operators import DraftTreeAttention
    B, T, nh, hd = s["q"].shape
    op = DraftTreeAttention(batch=B, nodes=T, max_ctx=s["max_ctx"], num_kv_groups=s["nkv"],
                            q_heads_per_group=nh // s["nkv"], head_dim=hd, dtype=s["q"].dtype)
    op(s["q"], s["k_cache"], s["v_cache"], s["k_draft"], s["v_draft"], s["ctx_len"], s["mask"], s["out"],
       num_nodes=s["num_nodes"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _commit_plain(s):
    L, B, nkv, max_ctx, hd = s["k_caches"].shape
    T = s["tokens"].shape[1]
    dev = s["tokens"].device
    node = torch.arange(T, device=dev)[None]
    rows = torch.arange(B, device=dev)
    live = node < s["num_nodes"][:, None]
    cur = torch.zeros(B, dtype=torch.int64, device=dev)
    going = torch.ones(B, dtype=torch.bool, device=dev)
    path = torch.full((B, T), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    for d in range(1, T):                                                                  # one level of the tree
        want = s["predicted"][rows, cur]
        fits = live & (node > cur[:, None]) & (s["parents"] == cur[:, None]) & (s["tokens"] == want[:, None])
        going = going & fits.any(1) & (s["ctx_len"] + d < max_ctx)
        cur = torch.where(going, fits.int().argmax(1), cur)
        path[:, d] = torch.where(going, cur, -1).int()
    count = (path >= 0).sum(1).int()
    b, i = torch.nonzero(path >= 0, as_tuple=True)
    at, src = s["ctx_len"][b] + i, path[b, i].long()
    s["k_caches"][:, b, :, at] = s["k_drafts"][:, b, src].transpose(0, 1)
    s["v_caches"][:, b, :, at] = s["v_drafts"][:, b, src].transpose(0, 1)
    return {"path": path, "num_accepted": count, "next_token": s["predicted"][rows, cur], "new_len": s["ctx_len"] + count,
            "k": s["k_caches"], "v": s["v_caches"]}


def _commit_own(s):
    from torch2iron_b200.operators import DraftTreeCommit
    L, B, nkv, max_ctx, hd = s["k_caches"].shape
    op = DraftTreeCommit(layers=L, batch=B, nodes=s["tokens"].shape[1], max_ctx=max_ctx, num_kv_groups=nkv,
                         head_dim=hd, dtype=s["k_caches"].dtype)
    op(s["tokens"], s["parents"], s["predicted"], s["ctx_len"], s["k_drafts"], s["v_drafts"], s["k_caches"],
       s["v_caches"], s["path"], s["num_accepted"], s["next_token"], s["new_len"], num_nodes=s["num_nodes"])
    return {"path": s["path"], "num_accepted": s["num_accepted"], "next_token": s["next_token"],
            "new_len": s["new_len"], "k": s["k_caches"], "v": s["v_caches"]}


def _logprobs_plain(s):
    x = s["logits"].float()
    K = s["case"]["top"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    log_sum = torch.log(e.sum(1, keepdim=True))
    spread = torch.where(e > 0, e * (x - m), 0.0).sum(1) / e.sum(1)
    got = {"logprob": (x.gather(1, s["tokens"].long()[:, None]) - m - log_sum)[:, 0],
           "entropy": log_sum[:, 0] - spread}
    if K:
        top, index = torch.sort(x, dim=1, descending=True, stable=True)                    # ties: lowest index first
        got.update(top_logprob=top[:, :K] - m - log_sum, top_index=index[:, :K].int())
    return got


def _logprobs_own(s):
    from torch2iron_b200.operators import TokenLogProbs
    M, V = s["logits"].shape
    K = s["case"]["top"]
    op = TokenLogProbs(rows=M, vocab=V, num_top=K, dtype=s["logits"].dtype)
    op(s["logits"], s["tokens"], s["logprob"], entropy=s["entropy"], top_logprob=s["top_logprob"],
       top_index=s["top_index"])
    got = {"logprob": s["logprob"], "entropy": s["entropy"]}
    if K:
        got.update(top_logprob=s["top_logprob"], top_index=s["top_index"])
    return got


_run_plain = {"packed": _packed_plain, "tree": _tree_plain, "commit": _commit_plain, "logprobs": _logprobs_plain}
_run_own = {"packed": _packed_own, "tree": _tree_own, "commit": _commit_own, "logprobs": _logprobs_own}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    op = case["op"]
    if op == "logprobs":
        M, V, K = case["rows"], case["vocab"], case["top"]
        return {"bytes": M * V * size + M * (4 + 8 + 8 * K), "flops": 6 * M * V}
    nh, nkv, hd = HEADS[case["heads"]]
    if op == "packed":
        n, pre = _lengths(case), _prefixes(case)
        pairs = sum(a * p + a * (a + 1) // 2 for a, p in zip(n, pre))
        keys = sum(n) + sum(pre)
        return {"bytes": sum(n) * nh * (2 * hd * size + 4) + 2 * keys * nkv * hd * size, "flops": 4 * hd * nh * pairs}
    if op == "tree":
        live, ctx = _nodes(case), _contexts(case)
        pairs = sum(a * (c + 1) for a, c in zip(live, ctx))
        rows = sum(live)
        return {"bytes": rows * nh * (2 * hd * size + 4) + 2 * (sum(ctx) + rows) * nkv * hd * size,
                "flops": 4 * hd * nh * pairs}
    take = sum(_accepted(case))
    return {"bytes": take * case["layers"] * nkv * hd * size * 4 + 4 * case["rows"] * (4 * case["nodes"] + 5),
            "flops": 0}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "packed":
        out, lse = s["out"].double(), s["lse"].double()
        group = s["nh"] // s["nkv"]
        at = 0
        for b, (n, m) in enumerate(zip(s["n"], s["k_n"])):
            for h in range(s["nh"]):
                g = h // group
                k, v = ((s[x][at:at + n, g] if s["max_ctx"] is None else s[x][b, g, :m]).double() for x in ("k", "v"))
                for c in range(0, n, 2048):
                    e = min(n, c + 2048)
                    z = s["q"][at + c:at + e, h].double() @ k[:m - n + e].t() / math.sqrt(s["hd"])
                    later = torch.ones_like(z, dtype=torch.bool).triu_(m - n + c + 1)
                    z.masked_fill_(later, -math.inf)
                    top = torch.logsumexp(z, 1)
                    out[at + c:at + e, h] = torch.exp(z - top[:, None]) @ v[:m - n + e]
                    lse[at + c:at + e, h] = top
            at += n
        return {"out": out, "lse": lse}
    if op == "tree":
        out, lse = s["out"].double(), s["lse"].double()
        group = s["nh"] // s["nkv"]
        mask = s["mask"].cpu().numpy().view(np.uint64)
        for b, (n, c) in enumerate(zip(s["live"], s["ctx"])):
            sees = torch.tensor([[bool(mask[b, i, j // 64] >> np.uint64(j % 64) & np.uint64(1)) for j in range(n)]
                                 for i in range(n)], device=out.device)
            for g in range(s["nkv"]):
                k, v = (torch.cat([s[x + "_cache"][b, g, :c], s[x + "_draft"][b, :n, g]]).double() for x in ("k", "v"))
                q = s["q"][b, :n, g * group:(g + 1) * group].double()
                z = torch.einsum("ihd,jd->ihj", q, k) / math.sqrt(s["hd"])
                z[:, :, c:] = torch.where(sees[:, None], z[:, :, c:], -math.inf)
                top = torch.logsumexp(z, 2)
                out[b, :n, g * group:(g + 1) * group] = torch.einsum("ihj,jd->ihd", torch.exp(z - top[..., None]), v)
                lse[b, :n, g * group:(g + 1) * group] = top
        return {"out": out, "lse": lse}
    if op == "commit":
        tokens, parents, predicted = (s[x].tolist() for x in ("tokens", "parents", "predicted"))
        live, ctx = s["num_nodes"].tolist(), s["ctx_len"].tolist()
        T = case["nodes"]
        paths, nexts = [], []
        for b in range(case["rows"]):
            path = [0]
            while ctx[b] + len(path) < s["max_ctx"]:
                fits = [n for n in range(path[-1] + 1, live[b])
                        if parents[b][n] == path[-1] and tokens[b][n] == predicted[b][path[-1]]]
                if not fits:
                    break
                path.append(fits[0])
            for i, n in enumerate(path):
                for x in ("k", "v"):
                    s[x + "_caches"][:, b, :, ctx[b] + i] = s[x + "_drafts"][:, b, n]
            paths.append(path + [-1] * (T - len(path)))
            nexts.append(predicted[b][path[-1]])
        count = [sum(n >= 0 for n in p) for p in paths]
        as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=s["path"].device)  # noqa: E731
        return {"path": as_int(paths), "num_accepted": as_int(count), "next_token": as_int(nexts),
                "new_len": as_int([c + n for c, n in zip(ctx, count)]), "k": s["k_caches"], "v": s["v_caches"]}
    logprob, entropy, top, index = [], [], [], []
    K = case["top"]
    for x, t in zip(s["logits"], s["tokens"].tolist()):
        y = torch.log_softmax(x.double(), 0)
        logprob.append(y[t])
        entropy.append(-torch.special.xlogy(y.exp(), y.exp()).sum())
        if K:
            i = torch.sort(x, descending=True, stable=True).indices[:K]
            top.append(y[i])
            index.append(i.int())
    got = {"logprob": torch.stack(logprob), "entropy": torch.stack(entropy)}
    if K:
        got.update(top_logprob=torch.stack(top), top_index=torch.stack(index))
    return got
