"""The operators that check drafted tokens, as cases that can be timed and checked.

A case is a dict of plain values. `prepare` makes what a decoding program holds before the call, `run` is one pass through an
operator: with `own` as calls of the framework, without as elementary tensor operations in 32 bits. `exact` is the result from
the definition in 64 bits, `work` is the least a pass has to read, write and compute.

Kinds:

    attn      attention of a tree of drafted tokens over each sequence's cache (`ops.attn_tree`)
    append    rotation of the nodes' queries and keys by their depth, keys and values into the cache (`ops.rope_kv_append_tree`)
    keep      the greedy walk through a tree and the cache rows of the accepted nodes moved together (`ops.tree_accept`, `ops.kv_keep_path`)
    logprobs  log probabilities of given tokens, entropy and the best alternatives of rows of logits (`ops.token_logprobs`)

Sizes: 20 query and 5 key/value heads of 128, a vocabulary of 128256 and 30 layers is the 2B4T shape, 32 and 8 heads the wider one of
the benchmarks; up to 16 sequences is what a cache serves.
"""
from __future__ import annotations

import math

import torch

own = False

HEAD = 128     # size of an attention head
THETA = 500000.0


# ---- the cases ----------------------------------------------------------------------------------

def attn(b, t, heads, kv, length, dtype, ragged=False, name=""):
    return {"name": name, "kind": "attn", "b": b, "t": t, "heads": heads, "kv": kv, "length": length, "dtype": dtype, "ragged": ragged}


def append(b, t, heads, kv, length, ragged=False, name=""):
    return {"name": name, "kind": "append", "b": b, "t": t, "heads": heads, "kv": kv, "length": length, "ragged": ragged}


def keep(b, t, depth, kv, layers, length, name=""):
    return {"name": name, "kind": "keep", "b": b, "t": t, "depth": depth, "kv": kv, "layers": layers, "length": length}


def logprobs(rows, vocab, dtype, given, top, masked=False, pad=0, scale=1.0, name=""):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "given": given, "top": top, "masked": masked, "pad": pad,
            "scale": scale}


def listed() -> list:
    return [
        # a single token of one sequence with a short history: a draft of nothing, all latency
        attn(1, 1, 20, 5, 300, "f32", name="attn 1 x 1 node, 300 keys"),
        # a chain of five drafted tokens of one long chat
        attn(1, 5, 20, 5, 4001, "f32", name="attn 1 x 5 nodes, 4001 keys"),
        # trees of a batch of chats of all lengths, one of them without a draft
        attn(11, 26, 20, 5, 4000, "f32", ragged=True, name="attn 11 x 26 nodes, ragged"),
        # a wide tree of one sequence with a whole book behind it
        attn(1, 60, 32, 8, 65000, "bf16", name="attn 1 x 60 nodes, 65000 keys"),
        # the largest trees of a full cache
        attn(16, 64, 20, 5, 8100, "f32", name="attn 16 x 64 nodes, 8100 keys"),
        # the nodes of a short chain, and of full trees of a full cache
        append(1, 5, 20, 5, 700, name="append 1 x 5 nodes"),
        append(16, 61, 32, 8, 900, ragged=True, name="append 16 x 61 nodes"),
        # what a chain and what large trees leave in the cache
        keep(1, 6, 4, 5, 30, 700, name="keep 1 x 6 nodes"),
        keep(16, 64, 9, 5, 30, 400, name="keep 16 x 64 nodes"),
        # a generated token with a few alternatives
        logprobs(1, 128256, "f32", 1, 5, name="logprobs 1 row"),
        # the rows of a batch of draft trees, several candidates each, a vocabulary that is a multiple of nothing, some of it ruled out
        logprobs(203, 50021, "bf16", 4, 1, masked=True, scale=1.25, name="logprobs 203 rows bf16"),
        # a long prompt, scored token by token
        logprobs(2000, 128256, "f32", 1, 20, name="logprobs 2000 rows"),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng) -> dict:
    kind = rng.choice(["attn", "attn", "attn", "append", "keep", "logprobs", "logprobs"])
    heads, kv = rng.choice([(20, 5), (32, 8), (16, 4), (8, 8), (12, 2), (9, 1), (5, 5)])
    if kind == "attn":
        b, t = _log(rng, 1, 16), _log(rng, 1, 100)
        most = min(65000, int(1.0e10 / (b * t * heads * 128)), int(1.3e5 / b))
        c = attn(b, t, heads, kv, _log(rng, 1, max(2, most)), rng.choice(["f32", "bf16"]), rng.random() < 0.6)
    elif kind == "append":
        c = append(_log(rng, 1, 16), _log(rng, 1, 60), heads, kv, _log(rng, 1, 900), rng.random() < 0.5)
    elif kind == "keep":
        b, t = _log(rng, 1, 16), _log(rng, 2, 64)
        c = keep(b, t, rng.randint(1, min(t, 9)), rng.choice([1, 2, 4, 5]), rng.randint(1, 30), _log(rng, 1, 400))
    else:
        rows, vocab = _log(rng, 1, 2000), _log(rng, 100, 128256)
        c = logprobs(rows, vocab, rng.choice(["f32", "bf16"]), rng.randint(1, 8), rng.randint(0, 20), rng.random() < 0.4, rng.choice([0, 0, 3, 64]),
                     rng.choice([1.0, 1.0, 0.7, 1.5]))
    del c["name"]
    return c


def _lengths(case):
    """Committed positions of every sequence: all `length`, or spread below it."""
    b, n = case["b"], case["length"]
    return [n - (n * 3 * i) // (4 * b) if case.get("ragged") else n for i in range(b)]


def _counts(case):
    """Nodes in use of every sequence: all of them, or fewer, one sequence without any."""
    b, t = case["b"], case["t"]
    return [(0 if i == 2 else t - (5 * i) % t) if case.get("ragged") else t for i in range(b)]


def _kept(case):
    """How many nodes of every sequence are accepted."""
    return [1 + (case["depth"] - 1 + 3 * i) % case["depth"] for i in range(case["b"])]


# ---- what a program has in hand -----------------------------------------------------------------

def _random(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _parents(case, seed):
    """Trees: most nodes hang on one of the eight in front of them. Parents of every sequence, [b][t]."""
    g = torch.Generator().manual_seed(seed)
    b, t = case["b"], case["t"]
    back = 1 + (torch.rand(b, t, generator=g) * torch.arange(t).clamp(max=8)).long().clamp(max=7)
    return (torch.arange(t) - back).clamp(min=0).index_fill(1, torch.tensor([0]), -1).to(torch.int32)


def _cache(shape, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)


def prepare(case, seed) -> dict:
    g, s = _random(seed), {"kind": case["kind"]}
    on = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = 2.5 * torch.randn(rows, vocab + case["pad"], generator=g, device="cuda")
        if case["masked"]:
            x[:, :vocab][torch.rand(rows, vocab, generator=g, device="cuda") < 0.3] = -math.inf
        x = x.to(torch.float32 if case["dtype"] == "f32" else torch.bfloat16)
        s.update(logits=x[:, :vocab], tokens=torch.randint(0, vocab, (rows, case["given"]), generator=g, device="cuda", dtype=torch.int32), top=min(case["top"], vocab),
                 scale=case["scale"])
        return s
    b, t, kv, length = case["b"], case["t"], case["kv"], case["length"]
    cap = length + t + 3
    s.update(pos=on(_lengths(case)) if case["kind"] != "keep" else on([length] * b))
    if case["kind"] == "keep":
        cg = torch.Generator().manual_seed(seed)
        parents = _parents(case, seed)
        best = torch.randint(0, 1000, (b, t), generator=cg, dtype=torch.int32)
        tokens = torch.randint(1000, 2000, (b, t), generator=cg, dtype=torch.int32)   # drafts that miss
        for i, n in enumerate(_kept(case)):                                           # and a path that hits
            path = [0] + sorted((1 + torch.randperm(t - 1, generator=cg)[:n - 1]).tolist())
            for up, node in zip(path, path[1:]):
                parents[i, node], tokens[i, node] = up, best[i, up]
        s.update(parents=parents.cuda(), best=best.cuda(), tokens=tokens.cuda(), k=_cache((case["layers"], b, kv, cap, HEAD), g),
                 v=_cache((case["layers"], b, kv, cap, HEAD), g))
        return s
    s.update(parents=_parents(case, seed).cuda(), counts=on(_counts(case)) if case["ragged"] else None, most=max(_lengths(case)) + t, heads=case["heads"])
    s.update(k=_cache((b, kv, cap, HEAD), g), v=_cache((b, kv, cap, HEAD), g))
    q = torch.randn(b, t, case["heads"], HEAD, generator=g, device="cuda")
    if case["kind"] == "attn":
        s["q"] = (1.5 * q).to(torch.float32 if case["dtype"] == "f32" else torch.bfloat16)
        s["out"] = torch.zeros_like(s["q"])
        return s
    place = torch.arange(cap, dtype=torch.float64)[:, None] * THETA ** (-torch.arange(0, HEAD, 2, dtype=torch.float64) / HEAD)
    s.update(q=q, k_new=torch.randn(b, t, kv, HEAD, generator=g, device="cuda"), v_new=torch.randn(b, t, kv, HEAD, generator=g, device="cuda"),
             cos=torch.cos(place).repeat(1, 2).float().cuda(), sin=torch.sin(place).repeat(1, 2).float().cuda())
    return s


# ---- the plain form -----------------------------------------------------------------------------

def _ancestors(parents):
    """[b][t][t] truth values: node j is node i or one of its ancestors. Each product doubles the generations that are known."""
    t = parents.shape[1]
    known = (parents[:, :, None] == torch.arange(t, device=parents.device)).float() + torch.eye(t, device=parents.device)
    for _ in range(max(1, (t - 1).bit_length())):
        known = (known @ known).clamp(max=1.0)
    return known > 0.5


def _live(s):
    """[b][t]: the nodes in use."""
    b, t = s["parents"].shape
    at = torch.arange(t, device="cuda").expand(b, t)
    return at < s["counts"][:, None] if s["counts"] is not None else at >= 0


def _plain_attn(s):
    q, b, t, heads, most = s["q"], *s["parents"].shape, s["heads"], s["most"]
    kv = s["k"].shape[1]
    k, v = s["k"][:, :, :most].float(), s["v"][:, :, :most].float()
    node = torch.arange(most, device="cuda") - s["pos"][:, None]                      # which node a row of the cache holds
    inside = (node >= 0) & (node < t)
    seen = torch.gather(_ancestors(s["parents"]), 2, node.clamp(0, t - 1)[:, None].expand(b, t, most)) & inside[:, None] | (node < 0)[:, None]
    g = q.float().view(b, t, kv, heads // kv, HEAD).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, HEAD)
    scores = (g @ k.transpose(2, 3) / math.sqrt(HEAD)).view(b, kv, -1, t, most).masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = (e / e.sum(-1, keepdim=True)).view(b, kv, -1, most) @ v
    o = o.view(b, kv, heads // kv, t, HEAD).permute(0, 3, 1, 2, 4).reshape(b, t, heads, HEAD)
    s["out"].copy_(torch.where(_live(s)[:, :, None, None], o.to(q.dtype), s["out"]))
    return s["out"]


def _plain_append(s):
    b, t = s["parents"].shape
    live, half = _live(s), HEAD // 2
    depth = _ancestors(s["parents"]).sum(-1) - 1
    at = (s["pos"][:, None] + depth).long()
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    turned = lambda x: x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin  # noqa: E731
    s["q"].copy_(torch.where(live[:, :, None, None], turned(s["q"]), s["q"]))
    seq, row = torch.arange(b, device="cuda")[:, None].expand(b, t)[live], (s["pos"][:, None] + torch.arange(t, device="cuda"))[live]
    s["k"][seq, :, row] = turned(s["k_new"])[live].to(torch.bfloat16)
    s["v"][seq, :, row] = s["v_new"][live].to(torch.bfloat16)
    return s["q"], s["k"], s["v"]


def _plain_keep(s):
    parents, tokens, best = s["parents"].long(), s["tokens"], s["best"]
    b, t = parents.shape
    at = torch.arange(t, device="cuda")
    hit = (tokens == torch.gather(best, 1, parents.clamp(min=0))) & (parents >= 0)
    twin = (parents[:, :, None] == parents[:, None]) & hit[:, None] & (at[None, :] < at[:, None])   # a sibling in front hits too
    hit &= ~twin.any(-1)
    hit[:, 0] = True
    taken = (_ancestors(parents) & ~hit[:, None]).sum(-1) == 0
    count = taken.sum(-1)
    path = torch.where(taken, at, t).sort(-1).values
    last = torch.gather(path, 1, count[:, None] - 1)
    path = torch.where(at < count[:, None], path, -1)
    seq, place = torch.nonzero(path >= 0, as_tuple=True)
    to, come = s["pos"].long()[seq] + place, s["pos"].long()[seq] + path[seq, place]
    for c in (s["k"], s["v"]):
        c[:, seq, :, to] = c[:, seq, :, come]
    return path.int(), count.int(), torch.gather(best, 1, last)[:, 0], s["k"], s["v"]


def _plain_logprobs(s):
    x = s["logits"].float()
    c = x * s["scale"]
    top = c.amax(-1, keepdim=True)
    e = torch.exp(c - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    entropy = torch.where(e > 0, e * (lse - c), 0.0).sum(-1) / total[:, 0]
    best, ids = torch.sort(x, dim=-1, descending=True, stable=True)                  # the lower of equal ones first
    best, ids = best[:, :s["top"]], ids[:, :s["top"]].int()
    return torch.gather(c, 1, s["tokens"].long()) - lse, entropy, ids, best * s["scale"] - lse


def run(state):
    s, kind = state, state["kind"]
    if not own:
        return {"attn": _plain_attn, "append": _plain_append, "keep": _plain_keep, "logprobs": _plain_logprobs}[kind](s)
    from lemonade_burn_b200 import ops
    if kind == "attn":
        return ops.attn_tree(s["q"], s["k"], s["v"], s["pos"], s["parents"], s["counts"], out=s["out"])
    if kind == "append":
        ops.rope_kv_append_tree(s["q"], s["k_new"], s["v_new"], s["cos"], s["sin"], s["pos"], s["parents"], s["k"], s["v"], s["counts"])
        return s["q"], s["k"], s["v"]
    if kind == "keep":
        path, count, after = ops.tree_accept(s["tokens"], s["parents"], s["best"])
        ops.kv_keep_path(s["k"], s["v"], s["pos"], path, count)
        return path, count, after, s["k"], s["v"]
    got = ops.token_logprobs(s["logits"], s["tokens"], s["top"], s["scale"])
    return got.logprobs, got.entropy, got.top_ids, got.top_logprobs


# ---- the least work -----------------------------------------------------------------------------

def work(case) -> dict:
    kind = case["kind"]
    if kind == "logprobs":
        n, size = case["rows"] * case["vocab"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": n * size + case["rows"] * (8 * case["given"] + 8 * case["top"] + 4), "flops": 5 * n}
    counts, kv = _counts(case), case["kv"]
    if kind == "keep":
        moved = sum(n - 1 for n in _kept(case))   # node 0 lies where it belongs
        return {"bytes": moved * case["layers"] * kv * HEAD * 2 * 2 * 2 + case["b"] * case["t"] * 16, "flops": case["b"] * case["t"]}
    nodes, heads = sum(counts), case["heads"]
    if kind == "append":
        return {"bytes": nodes * HEAD * (8 * heads + 2 * 6 * kv + 8), "flops": nodes * HEAD * 3 * (heads + kv)}
    size = 4 if case["dtype"] == "f32" else 2
    keys = [n + c if c else 0 for n, c in zip(_lengths(case), counts)]
    return {"bytes": sum(keys) * kv * HEAD * 4 + 2 * nodes * heads * HEAD * size, "flops": sum(4 * n * c for n, c in zip(keys, counts)) * heads * HEAD}


# ---- the same from the definition, in 64 bits ---------------------------------------------------

def _chain(parents, i):
    """Node i and its ancestors."""
    found = []
    while i >= 0:
        found.append(i)
        i = parents[i]
    return found


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "logprobs":
        lp, entropy, ids, best = [], [], [], []
        for x, tokens in zip(s["logits"].split(64), s["tokens"].split(64)):
            d = x.double() * s["scale"]
            logp = torch.log_softmax(d, -1)
            lp.append(torch.gather(logp, 1, tokens.long()))
            entropy.append(torch.special.entr(logp.exp()).sum(-1))
            # a total order of (value, place): what is larger, then what comes first
            order = torch.sort(-x.double(), dim=-1, stable=True).indices[:, :s["top"]]
            ids.append(order.int())
            best.append(torch.gather(logp, 1, order))
        return torch.cat(lp), torch.cat(entropy), torch.cat(ids), torch.cat(best)
    parents, pos = s["parents"].tolist(), s["pos"].tolist()
    if kind == "keep":
        b, t = len(parents), len(parents[0])
        tokens, best = s["tokens"].tolist(), s["best"].tolist()
        paths, after = [], []
        for i in range(b):
            path = [0]
            while True:
                nodes = [n for n in range(t) if parents[i][n] == path[-1] and tokens[i][n] == best[i][path[-1]]]
                if not nodes:
                    break
                path.append(nodes[0])
            rows = torch.tensor([pos[i] + n for n in path], device="cuda")
            for c in (s["k"], s["v"]):
                c[:, i, :, pos[i]:pos[i] + len(path)] = c[:, i].index_select(2, rows)
            paths.append(path + [-1] * (t - len(path)))
            after.append(best[i][path[-1]])
        count = [sum(n >= 0 for n in p) for p in paths]
        return torch.tensor(paths, dtype=torch.int32), torch.tensor(count, dtype=torch.int32), torch.tensor(after, dtype=torch.int32), s["k"], s["v"]
    counts, heads = _counts(case), case["heads"]
    if kind == "append":
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        for i, n in enumerate(counts):
            for node in range(n):
                at = pos[i] + len(_chain(parents[i], node)) - 1
                c, sn = s["cos"][at, :64].double(), s["sin"][at, :64].double()
                a, b = q[i, node, :, :64].clone(), q[i, node, :, 64:].clone()
                q[i, node, :, :64], q[i, node, :, 64:] = a * c - b * sn, b * c + a * sn
                a, b = s["k_new"][i, node].double().split(64, -1)
                k[i, :, pos[i] + node] = torch.cat([a * c - b * sn, b * c + a * sn], -1)
                v[i, :, pos[i] + node] = s["v_new"][i, node].double()
        return q, k, v
    out = s["out"].double()
    share = heads // case["kv"]
    for i, n in enumerate(counts):
        if not n:
            continue
        rows = pos[i] + n
        unseen = torch.full((n, n), True)
        for node in range(n):
            unseen[node, _chain(parents[i], node)] = False
        for h in range(heads):
            k, v = s["k"][i, h // share, :rows].double(), s["v"][i, h // share, :rows].double()
            scores = s["q"][i, :n, h].double() @ k.T / math.sqrt(HEAD)
            scores[:, pos[i]:][unseen.cuda()] = -math.inf
            out[i, :n, h] = torch.softmax(scores, -1) @ v
    return out
