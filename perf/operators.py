"""The work that is timed for the operators of speculative decoding: attention for trees of drafted tokens over the paged
cache, sampling with a least share of the most likely token's probability (min-p) from given random numbers, the walk that
takes the drafted tokens that the model agrees with, and the move of their keys and values to where they belong.

`listed()` names the cases, `draw(rng)` gives another one of the same ranges, `prepare` makes what a program holds before the
call, `run` is one pass, `work` what a pass cannot do without, and `exact` the same outputs in 64 bits.  With `own` set `run`
calls the framework, without it the plain form: elementary tensor operations in 32 bits (64 where a border decides).

A request's drafted tokens are a tree of at most 64 nodes, a parent before its children; node 0 is the token sampled last.
Node i of a request with `before` tokens in its cache has its key and value at place before + i and stands at position
before + depth(i); it sees every earlier token (or those within the window) and, among the nodes, those whose bits its
`visible` number has.
"""
from __future__ import annotations

import math
import random
import zlib

import numpy as np
import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# --------------------------------------------------------------------------------------------------------------- cases
def _tree(name, requests, nodes, before, heads, kv_heads, hd, page=16, dtype="bf16", window=0):
    """nodes, before: (least, most) of a request; the first request has the most of both."""
    return {"name": name, "op": "tree", "requests": requests, "nodes_low": nodes[0], "nodes": nodes[1], "before_low": before[0],
            "before": before[1], "heads": heads, "kv_heads": kv_heads, "hd": hd, "page": page, "dtype": dtype, "window": window}


def _sample(name, rows, vocab, temperature, top_k, top_p, min_p, spread=2.5):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k, "top_p": top_p,
            "min_p": min_p, "spread": spread}


def _accept(name, requests, chains, length):
    return {"name": name, "op": "accept", "requests": requests, "chains": chains, "length": length}


def _keep(name, requests, chains, length, slabs, kv_heads, hd, before, page=16, dtype="bf16"):
    return {"name": name, "op": "keep", "requests": requests, "chains": chains, "length": length, "slabs": slabs, "kv_heads": kv_heads, "hd": hd,
            "before": before, "page": page, "dtype": dtype}


def listed():
    return [
        # one user's eight drafted tokens behind a short conversation, a layer of the 0.5B sizes: latency
        _tree("tree_one_user_8_nodes", 1, (8, 8), (301, 301), 14, 2, 64),
        # eight users, 16 nodes each, behind 2,048 tokens, a layer of the 1.5B sizes: what a drafting server runs most
        _tree("tree_8_users_16_nodes", 8, (16, 16), (1900, 2048), 12, 2, 128),
        # a busy server, users with few and many drafted tokens behind short and long contexts, a layer of the 0.5B sizes
        _tree("tree_64_users_ragged", 64, (1, 32), (128, 4001), 14, 2, 64),
        # whole trees behind long documents, a layer of the 7B sizes
        _tree("tree_2_users_64_nodes_long", 2, (64, 64), (30000, 32001), 28, 4, 128),
        # the 32-bit path, three users behind 500 to 1,021 tokens
        _tree("tree_3_users_f32", 3, (5, 12), (500, 1021), 14, 2, 64, dtype="f32"),
        # one user's next token, min-p alone, over the 151,936 tokens of the 0.5B sizes
        _sample("sample_one_min_p", 1, 151936, 1.0, 0, 1.0, 0.05),
        # a batch with all three cuts at the command line's other settings
        _sample("sample_64_all_cuts", 64, 151936, 0.8, 50, 0.95, 0.1),
        # every node of 64 users' trees at a vocabulary of 32,768, min-p behind top-p
        _sample("sample_1024_nodes_top_p_min_p", 1024, 32768, 0.7, 0, 0.9, 0.02),
        # the walk: one user's chain of eight, and 256 users with four chains of 15 each
        _accept("accept_one_user", 1, 1, 7),
        _accept("accept_256_users", 256, 4, 15),
        # the accepted tokens' keys and values in all layers: one user at the 0.5B sizes, 64 users at the 1.5B sizes
        _keep("keep_one_user", 1, 3, 5, 24, 2, 64, 301),
        _keep("keep_64_users", 64, 4, 15, 28, 2, 128, 203),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "sample", "sample", "accept", "keep"])
    if op == "tree":
        heads, kv_heads = rng.choice([(14, 2), (12, 2), (16, 2), (28, 4), (4, 2), (3, 1), (8, 8), (40, 8), (16, 1)])
        hd = rng.choice([64, 128, 64, 128, 16, 32, 48, 80, 96, 256])
        requests, nodes = _log(rng, 1, 64), _log(rng, 1, 64)
        # (no more than the largest listed case has: keys times rows, and keys)
        most = min(32000, int(2 * 64 * 28 * 32000 * 128 / (requests * nodes * heads * hd)), int(2 * 4 * 32000 * 128 / (requests * kv_heads * hd)))
        before = _log(rng, 1, max(most, 2)) - 1
        case = _tree(None, requests, (rng.randint(1, nodes), nodes), (rng.randint(0, before), before), heads, kv_heads, hd,
                     rng.choice([16, 16, 16, 32, 48, 64]), rng.choice(["bf16", "bf16", "f32"]), rng.choice([0, 0, 0, _log(rng, 1, 4000)]))
    elif op == "sample":
        rows = _log(rng, 1, 256)
        vocab = _log(rng, 2, min(152064, 64 * 151936 // rows))
        case = _sample(None, rows, vocab, rng.choice([0.3, 0.7, 0.8, 1.0, 1.5]), rng.choice([0, 0, 1, 20, 50, 200]),
                       rng.choice([1.0, 1.0, 0.5, 0.9, 0.95]), rng.choice([0.0, 0.01, 0.05, 0.1, 0.5]), rng.choice([1.0, 2.5, 4.0]))
    elif op == "accept":
        chains = rng.randint(1, 6)
        case = _accept(None, _log(rng, 1, 256), chains, rng.randint(1, 63 // chains))
    else:
        chains = rng.randint(1, 6)
        case = _keep(None, _log(rng, 1, 64), chains, rng.randint(1, min(15, 63 // chains)), rng.randint(1, 28), rng.choice([1, 2, 4]),
                     rng.choice([16, 64, 80, 128]), _log(rng, 1, 203), rng.choice([16, 32, 48]), rng.choice(["bf16", "bf16", "f32"]))
    del case["name"]
    return case


# -------------------------------------------------------------------------------------------------------------- inputs
def _sizes(case):
    """Nodes and earlier tokens of every request: the sizes belong to the case, whatever the seed of the inputs."""
    rng = random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    if "chains" in case:
        n = [1 + case["chains"] * case["length"]] * case["requests"]
        return n, [max(0, case.get("before", 0) - rng.randint(0, 40)) for _ in n]
    n = [case["nodes"]] + [rng.randint(case["nodes_low"], case["nodes"]) for _ in range(case["requests"] - 1)]
    b = [case["before"]] + [rng.randint(case["before_low"], case["before"]) for _ in range(case["requests"] - 1)]
    return n, b


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _normal(shape, g, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _tables(n, before, page, rng):
    """Block tables of pages in no order, as a server that has run for a while has them; and the number of pages."""
    need = [-(-(a + b) // page) for a, b in zip(n, before)]
    ids = list(range(sum(need) + 3))
    rng.shuffle(ids)
    width = max(need)
    rows, at = [], 0
    for k in need:
        rows.append(ids[at : at + k] + [-1] * (width - k))
        at += k
    return _ints(rows), sum(need) + 3


def _starts(n):
    return [sum(n[:i]) for i in range(len(n))]


def _depths_and_masks(parents):
    """Of one request's tree: every node's depth, and the bits of its ancestors and itself, as signed 64-bit numbers."""
    depth, mask = [], []
    for i, p in enumerate(parents):
        depth.append(depth[p] + 1 if p >= 0 else 0)
        mask.append((mask[p] if p >= 0 else 0) | 1 << i)
    return depth, [m - (1 << 64) if m >> 63 else m for m in mask]


def _walk_inputs(case, rng, n):
    """Chains of drafted tokens behind the root, and what the model's sampler says after each node: it follows one chain for
    some of its length, as a model does whose text the drafts foresee in part."""
    tokens, parents, sampled = [], [], []
    for _ in n:
        tok, par, sam = [rng.randrange(151936)], [-1], [rng.randrange(151936)]
        for _ in range(case["chains"]):
            for i in range(case["length"]):
                par.append(0 if i == 0 else len(par) - 1)
                tok.append(rng.randrange(151936))
                sam.append(rng.randrange(151936))
        chain, agrees = rng.randrange(case["chains"]), rng.randint(0, case["length"])
        for i in range(agrees):
            node = 1 + chain * case["length"] + i
            sam[par[node]] = tok[node]
        tokens += tok
        parents += par
        sampled += sam
    return tokens, parents, sampled


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + zlib.crc32(repr(sorted(case.items(), key=lambda kv: kv[0])).encode()))
    rng = random.Random(int(seed) * 7919 + 1)
    s = dict(case)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a few tokens stand out above many that hardly count, as a trained model's logits do
        x = torch.randn((rows, vocab), generator=g, device=DEV) * case["spread"]
        x += 6.0 * (torch.rand((rows, vocab), generator=g, device=DEV) < 20.0 / vocab)
        s.update(logits=x, temperatures=torch.full((rows,), case["temperature"], device=DEV), top_ks=_ints([case["top_k"]] * rows),
                 top_ps=torch.full((rows,), case["top_p"], device=DEV), min_ps=torch.full((rows,), case["min_p"], device=DEV),
                 uniform=torch.randint(0, 1 << 24, (rows,), generator=g, device=DEV).float() / float(1 << 24))
        return s
    n, before = _sizes(case)
    s.update(n=n, q_start=_ints(_starts(n)), q_len=_ints(n), max_q_len=max(n), tokens_in_all=sum(n))
    if case["op"] == "tree":
        dt, hq, hk, hd, page = TYPES[case["dtype"]], case["heads"], case["kv_heads"], case["hd"], case["page"]
        tables, pages = _tables(n, before, page, rng)
        positions, visible = [], []
        for a, b in zip(n, before):
            depth, mask = _depths_and_masks([-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, a)])
            positions += [b + d for d in depth]
            visible += mask
        kv = [a + b for a, b in zip(n, before)]
        s.update(qkv=_normal((sum(n), (hq + 2 * hk) * hd), g, dt, 1.5), k_cache=_normal((pages, hk, page, hd), g, dt),
                 v_cache=_normal((pages, hk, hd, page), g, dt), tables=tables, kv_len=_ints(kv), max_kv_len=max(kv),
                 positions=_ints(positions), visible=_ints(visible, torch.int64), scale=hd ** -0.5)
        return s
    tokens, parents, sampled = _walk_inputs(case, rng, n)
    s.update(tokens=_ints(tokens), parents=_ints(parents), sampled=_ints(sampled))
    if case["op"] == "accept":
        s["visible"] = _ints([m for a, at in zip(n, _starts(n)) for m in _depths_and_masks(parents[at : at + a])[1]], torch.int64)
        return s
    paths = []
    for a, at in zip(n, _starts(n)):                       # the accepted nodes, -1 behind the last
        path = [0]
        while True:
            nxt = [i for i in range(path[-1] + 1, a) if parents[at + i] == path[-1] and tokens[at + i] == sampled[at + path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        paths.append(path + [-1] * (64 - len(path)))
    dt, hk, hd, page = TYPES[case["dtype"]], case["kv_heads"], case["hd"], case["page"]
    tables, pages = _tables(n, before, page, rng)
    s.update(k_cache=_normal((case["slabs"], pages, hk, page, hd), g, dt), v_cache=_normal((case["slabs"], pages, hk, hd, page), g, dt), tables=tables,
             before_all=_ints(before), path=_ints(paths), count=_ints([sum(p >= 0 for p in q) for q in paths]))
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_tree(s):
    """Softmax attention of every node over its request's earlier tokens and the nodes that it sees: 32 bits, rounded once."""
    hq, hk, hd, page, nodes = s["heads"], s["kv_heads"], s["hd"], s["page"], s["max_q_len"]
    b, width = s["tables"].shape
    group, keys = hq // hk, width * page
    i = torch.arange(nodes, device=DEV)
    there = i[None] < s["q_len"][:, None]                                                   # [B, N]
    rows = (s["q_start"][:, None] + i[None]).clamp(max=s["qkv"].shape[0] - 1).long()
    q = s["qkv"].float()[rows][..., : hq * hd].reshape(b, nodes, hk, group, hd).permute(0, 2, 1, 3, 4).reshape(b, hk, nodes * group, hd)
    at = s["tables"].clamp(min=0).long()
    k = s["k_cache"][at].float().permute(0, 2, 1, 3, 4).reshape(b, hk, keys, hd)
    v = s["v_cache"][at].float().permute(0, 2, 1, 4, 3).reshape(b, hk, keys, hd)
    j = torch.arange(keys, device=DEV)
    before = (s["kv_len"] - s["q_len"])[:, None]
    node = (j[None] - before)                                                               # [B, L]: which node a key belongs to
    bits = (s["visible"][rows][:, :, None] >> node.clamp(0, 63)[:, None]) & 1
    early = (node < 0)[:, None].expand(b, nodes, keys)
    if s["window"] > 0:
        early = early & (j[None, None] > s["positions"][rows][:, :, None] - s["window"])
    sees = early | ((bits != 0) & (node >= 0)[:, None] & (j[None] < s["kv_len"][:, None])[:, None])
    score = torch.matmul(q, k.transpose(2, 3)) * s["scale"]                                  # [B, Hk, N * G, L]
    score = score.view(b, hk, nodes, group, keys).masked_fill(~sees[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hk, nodes * group, keys), v.masked_fill((j[None] >= s["kv_len"][:, None])[:, None, :, None], 0.0))
    o = o.view(b, hk, nodes, group, hd) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 2, 1, 3, 4).reshape(b, nodes, hq * hd)
    return o[there].to(s["qkv"].dtype)


def _plain_sample(s):
    """What top-k and top-p keep (ties at a border whole), of that the tokens at least min_p times as likely as the most likely, and the
    first of those in index order whose running sum passes uniform * their sum.  64 bits: every cut is a border."""
    x, vocab = s["logits"], s["vocab"]
    w = torch.exp((x - x.amax(1, keepdim=True)).double() / s["temperatures"][:, None].double())
    best = torch.sort(w, dim=1, descending=True).values
    k = s["top_k"] if 0 < s["top_k"] < vocab else vocab
    kept = w >= best[:, k - 1 : k]
    mass = torch.where(kept, w, torch.zeros_like(w)).sum(1, keepdim=True)
    if s["top_p"] < 1:
        above = torch.cumsum(best, 1) - best                                                # mass in front of each place
        first = torch.searchsorted(best.neg().contiguous(), w.neg().contiguous())           # the first place of this weight
        kept = kept & (torch.gather(above, 1, first) < mass * s["top_ps"][:, None].double())
    kept = kept & (w >= s["min_ps"][:, None].double())
    run_sum = torch.cumsum(torch.where(kept, w, torch.zeros_like(w)), 1)
    point = s["uniform"][:, None].double() * run_sum[:, -1:]
    return (kept & (run_sum > point)).int().argmax(1).int()


def _plain_accept(s):
    """A node is accepted if every node from the root to it is the lowest child of its parent whose token is what was sampled after that parent."""
    nodes, t = 64, s["tokens"].shape[0]
    b = s["q_len"].shape[0]
    i = torch.arange(nodes, device=DEV)
    there = i[None] < s["q_len"][:, None]
    rows = (s["q_start"][:, None] + i[None]).clamp(max=t - 1).long()
    tok, par, sam = s["tokens"][rows], s["parents"][rows].long(), s["sampled"][rows]
    agrees = there & (par >= 0) & (tok == torch.gather(sam, 1, par.clamp(min=0)))
    rival = agrees[:, None, :] & agrees[:, :, None] & (par[:, None, :] == par[:, :, None]) & (i[None, :] < i[:, None])[None]
    agrees = (agrees & ~rival.any(2)) | (i == 0)[None]
    ancestors = (s["visible"][rows][:, :, None] >> i) & 1
    accepted = there & ((ancestors == 0) | agrees[:, None, :]).all(2)
    count = accepted.sum(1)
    path = torch.where(accepted, i[None], nodes + i[None]).sort(1).values
    live = path < nodes
    out = torch.gather(sam, 1, path.clamp(max=nodes - 1))
    minus = torch.full_like(out, -1)
    return torch.where(live, path.int(), minus), count.int(), torch.where(live, out, minus)


def _plain_keep(s):
    """Key and value of the i-th accepted node go to place before + i, in every layer."""
    page = s["page"]
    i = torch.arange(s["path"].shape[1], device=DEV)
    live = i[None] < s["count"][:, None]
    to, of = (s["before_all"][:, None] + i[None]).long(), (s["before_all"][:, None] + s["path"]).long()
    b = torch.arange(to.shape[0], device=DEV)[:, None].expand_as(to)
    to, of, b = to[live], of[live], b[live]
    to_page, of_page = s["tables"][b, to // page].long(), s["tables"][b, of // page].long()
    s["k_cache"][:, to_page, :, to % page] = s["k_cache"][:, of_page, :, of % page]
    s["v_cache"][:, to_page, :, :, to % page] = s["v_cache"][:, of_page, :, :, of % page]
    return s["k_cache"], s["v_cache"]


def run(s):
    if own:
        import easy_gpt  # noqa: F401  (makes easy_gpt.cpp_amd importable)
        from easy_gpt.cpp_amd import kernels

        k = kernels.backend()
        if s["op"] == "tree":
            out = torch.empty((s["qkv"].shape[0], s["heads"] * s["hd"]), dtype=s["qkv"].dtype, device=DEV)
            k.tree_attention(s["qkv"], out, s["k_cache"], s["v_cache"], s["tables"], s["q_start"], s["q_len"], s["kv_len"], s["visible"],
                             s["heads"], s["kv_heads"], s["hd"], s["page"], s["scale"], s["max_q_len"], s["max_kv_len"], window=s["window"],
                             positions=s["positions"] if s["window"] else None)
            return out
        if s["op"] == "sample":
            out = torch.empty(s["rows"], dtype=torch.int32, device=DEV)
            k.sample(s["logits"], s["temperatures"], s["top_ks"], s["top_ps"], s["uniform"], out, min_p=s["min_ps"])
            return out
        if s["op"] == "accept":
            return k.accept_drafts(s["tokens"], s["parents"], s["sampled"], s["q_start"], s["q_len"])
        k.keep_drafts(s["k_cache"], s["v_cache"], s["tables"], s["before_all"], s["path"], s["count"])
        return s["k_cache"], s["v_cache"]
    if s["op"] == "tree":
        return _plain_tree(s)
    if s["op"] == "sample":
        return _plain_sample(s)
    return _plain_accept(s) if s["op"] == "accept" else _plain_keep(s)


# ----------------------------------------------------------------------------------------------------- floors and 64 bits
def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * 4 + 24), "flops": case["rows"] * case["vocab"] * 3}
    n, before = _sizes(case)
    if case["op"] == "tree":
        size, hq, hk, hd, window = TYPES[case["dtype"]].itemsize, case["heads"], case["kv_heads"], case["hd"], case["window"]
        reads = [a + (min(b, window) if window else b) for a, b in zip(n, before)]
        return {"bytes": size * hd * (2 * hk * sum(reads) + 2 * hq * sum(n)), "flops": 4 * hd * hq * sum(a * r for a, r in zip(n, reads))}
    if case["op"] == "accept":
        return {"bytes": 12 * sum(n) + 4 * len(n) * (2 * 64 + 3), "flops": sum(n)}
    # (half of a chain agrees on average, and one chain's tokens lie where they belong already)
    moved = case["requests"] * case["length"] / 2 * (1 - 1 / case["chains"])
    entry = 2 * case["slabs"] * case["kv_heads"] * case["hd"] * TYPES[case["dtype"]].itemsize
    return {"bytes": 2 * moved * entry + 4 * case["requests"] * (64 + 3), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tree":
        return _exact_tree(s)
    if case["op"] == "sample":
        return _exact_sample(s)
    n = s["n"]
    if case["op"] == "accept":
        tok, par, sam = s["tokens"].tolist(), s["parents"].tolist(), s["sampled"].tolist()
        paths, counts, outs = [], [], []
        for a, at in zip(n, _starts(n)):
            path, here = [0], 0
            while here is not None:
                wanted, here = sam[at + here], here
                here = next((i for i in range(here + 1, a) if par[at + i] == path[-1] and tok[at + i] == wanted), None)
                if here is not None:
                    path.append(here)
            paths.append(path + [-1] * (64 - len(path)))
            counts.append(len(path))
            outs.append([sam[at + i] for i in path] + [-1] * (64 - len(path)))
        return _ints(paths), _ints(counts), _ints(outs)
    k, v = s["k_cache"].double(), s["v_cache"].double()
    k0, v0 = k.clone(), v.clone()
    page, tables = s["page"], s["tables"].tolist()
    for r, (path, before) in enumerate(zip(s["path"].tolist(), s["before_all"].tolist())):
        for i, node in enumerate(path):
            if node > i:
                a, b = before + i, before + node
                k[:, tables[r][a // page], :, a % page] = k0[:, tables[r][b // page], :, b % page]
                v[:, tables[r][a // page], :, :, a % page] = v0[:, tables[r][b // page], :, :, b % page]
    return k, v


def _exact_tree(s):
    hq, hk, hd, page, out = s["heads"], s["kv_heads"], s["hd"], s["page"], []
    for r, (a, at, kv) in enumerate(zip(s["n"], _starts(s["n"]), s["kv_len"].tolist())):
        pages = s["tables"][r, : -(-kv // page)].long()
        k = s["k_cache"][pages].transpose(1, 2).reshape(-1, hk, hd)[:kv].double()             # [L, Hk, hd]
        v = s["v_cache"][pages].permute(0, 3, 1, 2).reshape(-1, hk, hd)[:kv].double()
        before = kv - a
        node = torch.arange(a, device=DEV)
        sees = torch.ones((a, kv), dtype=torch.bool, device=DEV)
        sees[:, before:] = (s["visible"][at : at + a, None] >> node & 1).bool()
        if s["window"]:
            sees[:, :before] = torch.arange(before, device=DEV) > s["positions"][at : at + a, None] - s["window"]
        q = s["qkv"][at : at + a, : hq * hd].double().view(a, hq, hd)
        o = torch.zeros((a, hq, hd), dtype=torch.float64, device=DEV)
        for h in range(hq):
            score = (q[:, h] @ k[:, h // (hq // hk)].t() * s["scale"]).masked_fill(~sees, -math.inf)
            o[:, h] = torch.where(sees.any(1, keepdim=True), torch.softmax(score, 1), torch.zeros_like(score)) @ v[:, h // (hq // hk)]
        out.append(o.view(a, hq * hd))
    return torch.cat(out)


def _exact_sample(s):
    x, picked = s["logits"].cpu().numpy().astype(np.float64), []
    t, p, m, u = (s[k].cpu().numpy().astype(np.float64) for k in ("temperatures", "top_ps", "min_ps", "uniform"))
    for r in range(s["rows"]):
        w = np.exp((x[r] - x[r].max()) / t[r])
        least = np.partition(w, -s["top_k"])[-s["top_k"]] if 0 < s["top_k"] < s["vocab"] else 0.0
        some = np.sort(w[w >= least])[::-1]
        if p[r] < 1:                                         # the weight with which the mass p is reached
            least = some[min(len(some) - 1, int(np.searchsorted(np.cumsum(some), p[r] * some.sum())))]
        kept = np.flatnonzero(w >= max(least, m[r]))
        mass = np.cumsum(w[kept])
        picked.append(int(kept[min(len(kept) - 1, int(np.searchsorted(mass, u[r] * mass[-1], side="right")))]))
    return _ints(picked)
